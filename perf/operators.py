"""The paged 8-bit KV cache at work, as cases to measure: rows of K and V
quantized as they are written, read back, and attended over.

The cache: pages of `page` tokens shared by all sequences, a block table per
sequence, one length per sequence; codes of one byte (e4m3 or int8) with an
fp32 scale for each `block` tokens of a KV head, a power of two.  The new
tokens of a sequence are its last ones: sequence b of length n holds its t_b
new tokens at positions n - t_b .. n - 1.

Sizes follow the package's constants and benchmark sweep (64 query heads over 8
KV heads of 128 channels, sinks of 4 tokens, windows up to 16384, contexts up
to 163840), its tests' other head groupings, and generic batch sizes.  Keys
carry a few channels far larger than the rest.
"""

import math
import os
import sys

import torch

own = False   # run(): the package's kernels instead of the plain form

D, SINK = 128, 4
SCALE = D**-0.5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LOWEST = -100   # least exponent of a scale


def _case(op, batch, length, tokens, code, dtype, page=64, block=32, layout="NHD", heads=64, kv_heads=8, even=False,
          window=0):
    """length: the longest sequence with its new tokens; tokens: most new
    tokens of a sequence; even: every sequence as long as the longest (else
    from short ones up to it); window: 0 = all tokens."""
    return dict(op=op, batch=batch, length=length, tokens=tokens, code=code, dtype=dtype, page=page, block=block,
                layout=layout, heads=heads, kv_heads=kv_heads, even=even, window=window)


def listed():
    return [
        # one user's token step: launch latency
        dict(_case("write", 1, 1000, 1, "e4m3", "bf16", page=16, block=16), name="write_e4m3_b1_token"),
        # a serving batch's token step, sequences of very different lengths
        dict(_case("write", 64, 16384, 1, "int8", "fp16", layout="HND"), name="write_int8_b64_token"),
        # a batch of prompts written whole, none of a round length but the longest
        dict(_case("write", 8, 8224, 8224, "e4m3", "bf16"), name="write_e4m3_b8_prompts"),
        # a short sequence read back (moved to another pool, or looked at)
        dict(_case("read", 1, 411, 411, "int8", "fp16", page=16, block=16), name="read_int8_b1_l411"),
        # a batch's caches read back for a kernel that wants whole rows
        dict(_case("read", 8, 16384, 16384, "e4m3", "bf16"), name="read_e4m3_b8_l16384"),
        # one user's token over a short context: launch latency
        dict(_case("attend", 1, 1000, 1, "e4m3", "fp16", page=16, block=16), name="attend_e4m3_b1_l1000"),
        # a batch over a long context: memory bandwidth
        dict(_case("attend", 32, 32768, 1, "e4m3", "fp16", even=True), name="attend_e4m3_b32_l32768"),
        # a serving batch of a bf16 model, small pages, lengths far apart
        dict(_case("attend", 16, 16384, 1, "int8", "bf16", page=16, block=16, layout="HND"),
             name="attend_int8_b16_l16384"),
        # sink and window over the longest context of the sweep
        dict(_case("attend", 8, 163840, 1, "int8", "fp16", page=128, block=128, even=True, window=4096),
             name="attend_int8_b8_w4096"),
        # drafted tokens checked at once
        dict(_case("attend", 8, 4000, 5, "e4m3", "bf16"), name="attend_e4m3_b8_draft5"),
        # a long prompt's last chunk over what is cached of it
        dict(_case("attend", 1, 8192, 2048, "e4m3", "bf16", even=True), name="attend_e4m3_chunk2048_l8192"),
        # prompts of many lengths, whole
        dict(_case("attend", 6, 3001, 3001, "int8", "fp16"), name="attend_int8_b6_prompts"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend"])
        heads, kv_heads = rng.choice([(64, 8), (64, 8), (64, 8), (32, 8), (32, 4), (16, 2), (8, 8), (12, 4), (16, 1)])
        page = rng.choice([16, 32, 64, 128])
        length = _log_int(rng, 8, 163840)
        if op == "read":
            tokens = length
        elif rng.random() < 0.5:
            tokens = 1
        else:
            tokens = rng.choice([rng.randint(2, 8), _log_int(rng, 2, 8192), length])
        c = _case(op, _log_int(rng, 1, 64), length, min(tokens, length), rng.choice(["e4m3", "int8"]),
                  rng.choice(["fp16", "bf16"] if op == "attend" else ["fp16", "bf16", "bf16", "fp32"]), page=page,
                  block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]), layout=rng.choice(["NHD", "HND"]),
                  heads=heads, kv_heads=kv_heads, even=rng.random() < 0.5,
                  window=_log_int(rng, 32, 16384) if op == "attend" and rng.random() < 0.3 else 0)
        # no dearer than the largest listed cases
        w = work(c)
        lens, new = _lens(c)
        pool = 2 * kv_heads * D * sum(lens)
        if w["bytes"] > (4.5e8 if op != "attend" else 2e9) or w["flops"] > 4.5e11 or pool > 2.7e9:
            continue
        if op == "attend":   # what the plain form holds of padded scores and of padded rows
            rows = _span(c) + SINK
            if c["batch"] * heads * max(new) * rows > 1.1e9 or c["batch"] * kv_heads * rows * D > 1.1e9:
                continue
        return c


# -- sizes --------------------------------------------------------------------

def _lens(c):
    """Lengths and new tokens of the sequences, on the host."""
    b = c["batch"]
    lens = [c["length"]] * b if c["even"] else [max(1, c["length"] * (i + 1) // b) for i in range(b)]
    new = [c["tokens"]] * b if c["even"] or c["tokens"] <= 8 else [max(1, c["tokens"] * (i + 1) // b) for i in range(b)]
    return lens, [min(t, n) for t, n in zip(new, lens)]


def _span(c):
    """Positions behind the sink that a sequence's new tokens attend at most."""
    return min(c["length"], c["window"] + max(_lens(c)[1]) - 1) if c["window"] else c["length"]


def _attended(c):
    """(tokens read, query-token pairs) of all sequences, for one head."""
    read = pairs = 0
    for n, t in zip(*_lens(c)):
        if not c["window"]:
            read, pairs = read + n, pairs + t * n - t * (t - 1) // 2
            continue
        first = max(0, n - t - c["window"] + 1)
        read += n - first + min(SINK, first)
        if t > 1:
            for i in range(t):
                lo = max(0, n - t + i - c["window"] + 1)
                pairs += n - t + i + 1 - lo + min(SINK, lo)
        else:
            pairs += n - first + min(SINK, first)
    return read, pairs


def work(c):
    kvh, new = c["kv_heads"], sum(_lens(c)[1])
    scales = 8 * kvh / c["block"]
    if c["op"] != "attend":
        return {"bytes": new * kvh * (2 * D * (BYTES[c["dtype"]] + 1)) + new * scales, "flops": 0.0}
    read, pairs = _attended(c)
    return {"bytes": 2 * new * c["heads"] * D * BYTES[c["dtype"]] + read * (2 * kvh * D + scales),
            "flops": 4.0 * D * c["heads"] * pairs}


# -- inputs -------------------------------------------------------------------

def _scale_of(amax, code):
    """The least power of two that brings amax into the codes' range."""
    m, e = torch.frexp(amax)
    e = e - 9 + (m > 0.875).int() if code == "e4m3" else e - 7 + (m > 127 / 128).int()
    e = torch.where(amax > 0, e, LOWEST).clamp(min=LOWEST)
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, code):
    """Values in the codes' range, rounded to codes (ties to even)."""
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _rows_first(pages, layout):
    """A pool as [page, row, head, channel]."""
    return pages if layout == "NHD" else pages.transpose(1, 2)


def _take(pages, *at):
    """Indexed rows of a pool, by their bytes."""
    return pages.view(torch.uint8)[at].view(pages.dtype)


def _put(pages, rows, *at):
    pages.view(torch.uint8)[at] = rows.view(torch.uint8)


def _pool(g, c, pages, far):
    """A pool of quantized values, and its scales; `far` channels are larger,
    and the blocks differ in magnitude."""
    p, block, kvh = c["page"], c["block"], c["kv_heads"]
    codes = torch.empty((pages, p, kvh, D) if c["layout"] == "NHD" else (pages, kvh, p, D), dtype=CODES[c["code"]],
                        device="cuda")
    scales = torch.empty((pages, kvh, p // block), device="cuda")
    step = max(1, (1 << 27) // (p * kvh * D))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = torch.randn((n, p // block, block, kvh, D), generator=g, device="cuda")
        x[..., far] *= 6
        x *= torch.exp2(0.5 * torch.randn((n, p // block, 1, kvh, 1), generator=g, device="cuda"))
        s = _scale_of(x.abs().amax((2, 4)), c["code"])
        scales[i:i + n] = s.transpose(1, 2)
        _rows_first(codes, c["layout"])[i:i + n] = _codes(x / s[:, :, None, :, None], c["code"]).view(n, p, kvh, D)
    return codes, scales


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    lens, new = _lens(c)
    order = torch.randperm(c["batch"], generator=g, device="cuda").tolist()
    lens, new = [lens[i] for i in order], [new[i] for i in order]
    blocks = [-(-n // c["page"]) for n in lens]
    total = sum(blocks) + 3   # some pages are free
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], max(blocks)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = perm[at:at + n]
        at += n
    far = torch.randperm(D, generator=g, device="cuda")[:3]
    k_pages, k_scales = _pool(g, c, total, far)
    v_pages, v_scales = _pool(g, c, total, far[:0])
    s = dict(c, k_pages=k_pages, v_pages=v_pages, k_scales=k_scales, v_scales=v_scales, table=table,
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), host_new=new, host_lens=lens,
             total=sum(new), most=max(new), longest=max(lens))
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    # one new token a sequence needs no offsets
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda") if c["tokens"] > 1 or c["op"] == "read" else None
    dt = DTYPES[c["dtype"]]
    if c["op"] == "write":
        k = torch.randn((s["total"], c["kv_heads"], D), generator=g, device="cuda")
        k[..., far] *= 6
        s["k"] = k.to(dt)
        s["v"] = torch.randn((s["total"], c["kv_heads"], D), generator=g, device="cuda", dtype=dt)
    elif c["op"] == "attend":
        s["q"] = torch.randn((s["total"], c["heads"], D), generator=g, device="cuda", dtype=dt)
    return s


# -- the plain form -----------------------------------------------------------

def _places(s):
    """Of every new token: its sequence, position, page and row."""
    n = torch.arange(s["total"], device="cuda")
    cu = s["cu"] if s["cu"] is not None else torch.arange(s["batch"] + 1, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], n, right=True)
    pos = s["lens"].long()[seq] - cu.long()[seq + 1] + n
    return cu.long(), seq, pos, s["table"].long()[seq, pos // s["page"]], pos % s["page"]


def _plain_write_one(s, x, pages, scales, cu, seq, pos, page, row):
    code, block = s["code"], s["block"]
    x = x.float()
    pages = _rows_first(pages, s["layout"])
    # the need of every block that the call writes to
    need = torch.zeros((scales.shape[0], scales.shape[2], scales.shape[1]), device="cuda")
    flat = need.view(-1, need.shape[2])
    which = page * need.shape[1] + row // block
    flat.scatter_reduce_(0, which[:, None].expand(-1, flat.shape[1]), x.abs().amax(-1), "amax")
    # a sequence's first block keeps the tokens before the call's
    first = cu[:-1]
    p0, r0 = page[first], row[first]
    b0 = r0 // block
    kept = r0 % block
    old = scales[p0, :, b0]
    want = _scale_of(flat[which[first]], code)
    grown = torch.where((kept > 0)[:, None], torch.maximum(old, want), want)
    rows = b0[:, None] * block + torch.arange(block, device="cuda")
    held = _take(pages, p0[:, None], rows)
    again = _codes(held.float() * (old / grown)[:, None, :, None], code)
    keep = (torch.arange(block, device="cuda") < kept[:, None])[:, :, None, None]
    _put(pages, torch.where(keep, again.view(torch.uint8), held.view(torch.uint8)), p0[:, None], rows)
    new = _scale_of(flat[which], code)
    mine = cu[seq]
    new = torch.where((which == which[mine])[:, None], grown[seq], new)
    scales[page, :, row // block] = new
    _put(pages, _codes(x / new[:, :, None], code), page, row)


def _plain_write(s):
    at = _places(s)
    _plain_write_one(s, s["k"], s["k_pages"], s["k_scales"], *at)
    _plain_write_one(s, s["v"], s["v_pages"], s["v_scales"], *at)
    return [s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]


def _values(s, pages, scales, page, row):
    """The rows' values in fp32: [..., KVH, D]."""
    return _take(_rows_first(pages, s["layout"]), page, row).float() * scales[page, :, row // s["block"]][..., None]


def _plain_read(s):
    _, _, _, page, row = _places(s)
    dt = DTYPES[s["dtype"]]
    return [_values(s, s["k_pages"], s["k_scales"], page, row).to(dt),
            _values(s, s["v_pages"], s["v_scales"], page, row).to(dt)]


def _plain_attend(s):
    cu, seq, pos, _, _ = _places(s)
    kvh, most, w = s["kv_heads"], s["most"], s["window"]
    lens = s["lens"].long()
    new = cu[1:] - cu[:-1]
    # the positions that a sequence's tokens may attend: the sink, then a span
    if w:
        start = (lens - new - w + 1).clamp(min=SINK)
        key = torch.cat([torch.arange(SINK, device="cuda").expand(len(lens), -1),
                         start[:, None] + torch.arange(_span(s), device="cuda")], 1)
    else:
        key = torch.arange(s["longest"], device="cuda").expand(len(lens), -1)
    inside = key < lens[:, None]
    key = torch.where(inside, key, 0)
    page, row = s["table"].long().gather(1, key // s["page"]), key % s["page"]
    kk = _values(s, s["k_pages"], s["k_scales"], page, row).permute(0, 2, 3, 1).contiguous()
    vv = _values(s, s["v_pages"], s["v_scales"], page, row).transpose(1, 2).contiguous()
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=s["total"] - 1)
    q = s["q"].float()[at].view(len(lens), most, kvh, -1, D).transpose(1, 2).reshape(len(lens), kvh, -1, D)
    mine = lens[:, None] - new[:, None] + i
    seen = inside[:, None] & (key[:, None] <= mine[:, :, None])
    if w:
        seen = seen & ((key[:, None] < SINK) | (key[:, None] > mine[:, :, None] - w))
    x = (q @ kk).mul_(SCALE).view(len(lens), kvh, most, -1, key.shape[1])
    x.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.view(len(lens), kvh, -1, key.shape[1]) @ vv
    o = o.view(len(lens), kvh, most, -1, D) / torch.where(total > 0, total, 1)
    o = o.transpose(1, 2).reshape(len(lens), most, -1, D)
    return o[seq, torch.arange(s["total"], device="cuda") - cu[seq]].to(s["q"].dtype)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "numerics-and-sparse-attn_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import paged8_kernel
    return paged8_kernel


def run(s):
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[s["op"]](s)
    p8 = _package()
    cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lens"])
    if s["op"] == "write":
        p8.write_paged8_cache(s["k"], s["v"], *cache, cu_seqlens=s["cu"], kv_layout=s["layout"])
        return [s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]
    if s["op"] == "read":
        k, v = p8.read_paged8_cache(*cache, cu_seqlens=s["cu"], num_tokens=s["total"], dtype=DTYPES[s["dtype"]],
                                    kv_layout=s["layout"])
        return [k, v]
    return p8.paged8_attention(s["q"], *cache, cu_seqlens=s["cu"], sm_scale=SCALE,
                               window=s["window"] or None, sink=SINK if s["window"] else 0, kv_layout=s["layout"])


# -- the definition in 64 bits ------------------------------------------------

def _held(s, b, first, end):
    """Page and row of positions first .. end - 1 of sequence b."""
    p = torch.arange(first, end, device="cuda")
    return s["table"][b].long()[p // s["page"]], p % s["page"]


def _in64(s, name, b, first, end):
    page, row = _held(s, b, first, end)
    x = _take(_rows_first(s[name + "_pages"], s["layout"]), page, row).double()
    return x * s[name + "_scales"].double()[page, :, row // s["block"]][..., None]


def _nearest64(x, code):
    if code == "int8":
        return torch.round(x)
    m, e = torch.frexp(x.abs())                       # e4m3: 3 bits behind the leading one, least exponent -6
    step = torch.exp2((torch.clamp(e - 1, min=-6) - 3).double())
    return torch.round(x / step) * step


def _exact_write(s, name):
    top = 448.0 if s["code"] == "e4m3" else 127.0
    codes = _rows_first(s[name + "_pages"], s["layout"]).double()
    scales, x = s[name + "_scales"].double(), s[name].double()
    block, at = s["block"], 0
    for b, (n, t) in enumerate(zip(s["host_lens"], s["host_new"])):
        pos = n - t
        while pos < n:
            # the blocks of a run of tokens, many whole ones at once
            many = 1 if pos % block or n - pos < block else (n - pos) // block
            end = min(n, (pos // block + many) * block)
            page, row = _held(s, b, pos, end)
            new = x[at:at + end - pos].view(many, -1, x.shape[1], D)
            amax = new.abs().amax((1, 3))
            e = torch.ceil(torch.log2(amax / top))
            e = torch.where(amax > top * torch.exp2(e), e + 1, e)
            e = torch.where(amax <= top * torch.exp2(e - 1), e - 1, e)
            sc = torch.exp2(torch.where(amax > 0, e, LOWEST).clamp(min=LOWEST))
            p, r = page.view(many, -1)[:, 0], row.view(many, -1)[:, 0]
            if pos % block:
                old = scales[p, :, r // block]
                sc = torch.maximum(old, sc)
                before, behind = _held(s, b, pos - pos % block, pos)
                codes[before, behind] = _nearest64(codes[before, behind] * (old / sc)[..., None], s["code"])
            codes[page, row] = _nearest64(new / sc[:, None, :, None], s["code"]).reshape(-1, x.shape[1], D)
            scales[p, :, r // block] = sc
            at, pos = at + end - pos, end
    return codes if s["layout"] == "NHD" else codes.transpose(1, 2).contiguous(), scales


def _exact_attend(s):
    out, at = [], 0
    for b, (n, t) in enumerate(zip(s["host_lens"], s["host_new"])):
        first = max(0, n - t - s["window"] + 1) if s["window"] else 0
        low = min(SINK, first)
        pos = torch.cat([torch.arange(low, device="cuda"), torch.arange(first, n, device="cuda")])
        kk = torch.cat([_in64(s, "k", b, 0, low), _in64(s, "k", b, first, n)])
        vv = torch.cat([_in64(s, "v", b, 0, low), _in64(s, "v", b, first, n)])
        mine = torch.arange(n - t, n, device="cuda")[:, None]
        seen = pos <= mine
        if s["window"]:
            seen &= (pos < SINK) | (pos > mine - s["window"])
        group = s["heads"] // s["kv_heads"]
        o = torch.empty((t, s["heads"], D), dtype=torch.float64, device="cuda")
        for h in range(s["heads"]):
            x = s["q"][at:at + t, h].double() @ kk[:, h // group].t().contiguous() * SCALE
            o[:, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ vv[:, h // group]
        out.append(o)
        at += t
    return torch.cat(out)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "write":
        k, v = _exact_write(s, "k"), _exact_write(s, "v")
        codes = [None, None] if c["code"] == "int8" else [k[0], v[0]]   # whole numbers: equal, or not
        return codes + [k[1], v[1]]
    if c["op"] == "read":
        return [torch.cat([_in64(s, x, b, 0, n) for b, n in enumerate(s["host_lens"])]) for x in "kv"]
    return _exact_attend(s)
