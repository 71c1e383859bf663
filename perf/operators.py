"""What the 4-bit key/value cache, its attention and the multi-axis rotary embedding are measured on.

Four operators of one path: queries and keys are rotated by positions on several axes (``kernels.rope_axes``), keys and
values are quantised into the pages of a 4-bit cache (``kv4.write``), read back from it (``kv4.read``) and attended
over in it (``kv4.attention``). ``run`` makes the framework's calls when ``own`` is true and computes the same in
elementary torch operations when it is false; ``exact`` states each operator in 64 bits.

Cache format (NVFP4, pages of one layer): codes uint8 [pages, kv_heads, page, D / 2], two E2M1 values a byte, the even
one in the low nibble; scales uint8 [pages, kv_heads, page, D / 16], one E4M3 byte per 16 values; a 32-bit factor
for the whole tensor. Position p of sequence b lives in page table[b, p // page], row p % page.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
AXES = {"image": (16, 56, 56), "video": (16, 24, 24), "small": (8, 12, 12), "plane": (32, 32)}


def _framework():
    folder = str(Path.cwd() / "qwen-image21-tensorfold-rtx_b200")
    if folder not in sys.path:
        sys.path.insert(1, folder)
    from tfimage import kernels, kv4

    return kernels, kv4


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of 8 sequences of a grouped-query model: 3 axes cut out of one frequency ladder (the two
        # halves of a head pair up), far text positions. Latency.
        dict(name="rope_token", op="rope", batch=8, n=1, hq=28, hk=4, dim=128, axes="video", sections=True,
             interleaved=False, norm=False, inverse=False, dtype="bf16", far=True),
        # The image tokens of one step of the synthetic MMDiT (64 x 64 grid, 24 heads x 128, axes 16/56/56), with the
        # block's q / k RMSNorm.
        dict(name="rope_image", op="rope", batch=1, n=4096, hq=24, hk=24, dim=128, axes="image", sections=False,
             interleaved=True, norm=True, inverse=False, dtype="bf16", far=False),
        # Gradient direction on a ragged video clip in 16 bits, narrow heads with a tail that is not rotated.
        dict(name="rope_video_back", op="rope", batch=2, n=10395, hq=16, hk=16, dim=80, axes="small", sections=False,
             interleaved=True, norm=False, inverse=True, dtype="fp16", far=False),
        # 13 sequences append one token each to short caches that are then read back whole. Latency.
        dict(name="kv4_append", op="write", batch=13, n=1, old=150, hk=8, dim=128, page=16, dtype="bf16"),
        # Prompts and reference images of 5 requests written at once and read back (24 heads, ragged).
        dict(name="kv4_prompts", op="write", batch=5, n=4352, old=0, hk=24, dim=128, page=64, dtype="bf16"),
        # A long context taken out of the cache whole, in 16 bits.
        dict(name="kv4_read_long", op="read", batch=3, n=50001, hk=8, dim=64, page=32, dtype="fp16"),
        # One query token over a short prompt, no shared heads: the smallest attention call. Latency.
        dict(name="decode_short", op="attention", batch=1, n=1, old=300, hq=24, hk=24, dim=128, page=64, dtype="bf16",
             causal=True, fresh=False, lse=False, ragged=False),
        # The decode step of a serving batch: 32 ragged sequences of up to 16384 tokens, 4 queries a key head.
        dict(name="decode_batch", op="attention", batch=32, n=1, old=16384, hq=32, hk=8, dim=128, page=64,
             dtype="bf16", causal=True, fresh=False, lse=False, ragged=True),
        # One sequence of 262143 tokens: the length has to be split.
        dict(name="decode_long", op="attention", batch=1, n=1, old=262143, hq=32, hk=4, dim=128, page=256,
             dtype="fp16", causal=True, fresh=False, lse=True, ragged=False),
        # Five drafted tokens of 6 sequences, the new keys still in 16 bits, narrow heads.
        dict(name="verify_draft", op="attention", batch=6, n=5, old=3001, hq=16, hk=2, dim=64, page=16, dtype="bf16",
             causal=True, fresh=True, lse=False, ragged=True),
        # The attention of one image block of the synthetic MMDiT: 4096 image tokens over the kept 256-token prompt in
        # 4 bits and their own keys in 16 bits.
        dict(name="image_step", op="attention", batch=1, n=4096, old=256, hq=24, hk=24, dim=128, page=64, dtype="bf16",
             causal=False, fresh=True, lse=False, ragged=False),
        # A chunk of a ragged prefill over long cached contexts, causal, grouped heads.
        dict(name="prefill_chunk", op="attention", batch=4, n=1500, old=9000, hq=16, hk=4, dim=128, page=128,
             dtype="fp16", causal=True, fresh=False, lse=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rope":
        axes, dim = rng.choice([("image", 128), ("video", 128), ("small", 64), ("small", 80), ("plane", 64)])
        batch, hk = _log(rng, 1, 8), rng.choice([2, 4, 8, 16, 24])
        hq = hk * rng.choice([1, 2, 4]) if hk < 16 else hk
        inverse = rng.random() < 0.3
        return dict(op=op, batch=batch, n=_log(rng, 1, max(1, 500_000 // (batch * (hq + hk)))), hq=hq, hk=hk, dim=dim,
                    axes=axes, sections=rng.random() < 0.4, interleaved=rng.random() < 0.6,
                    norm=not inverse and rng.random() < 0.5, inverse=inverse,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), far=rng.random() < 0.4)
    page, dim = rng.choice([16, 32, 64, 128, 256]), rng.choice([64, 128])
    if op in ("write", "read"):
        batch, hk = _log(rng, 1, 32), rng.choice([1, 2, 4, 8, 24])
        n = _log(rng, 1, max(2, 500_000 // (batch * hk)))
        if op == "read":
            return dict(op=op, batch=batch, n=n, hk=hk, dim=dim, page=page, dtype=rng.choice(["bf16", "fp16", "fp32"]))
        return dict(op=op, batch=batch, n=n, old=rng.choice([0, rng.randint(0, 500)]), hk=hk, dim=dim, page=page,
                    dtype=dtype)
    hk = rng.choice([1, 2, 4, 8, 24])
    hq = hk * rng.choice([1, 2, 4, 5, 8]) if hk < 24 else hk
    kind = rng.choice(["decode", "decode", "few", "many", "many"])
    batch = _log(rng, 1, 32) if kind != "many" else _log(rng, 1, 6)
    if kind == "many":  # pairs of query and key under half of the largest listed case's
        n = _log(rng, 33, max(34, min(4096, math.isqrt(200_000_000 // (batch * hq)))))
        old = _log(rng, 1, max(2, min(20000, 200_000_000 // (batch * n * hq))))
    else:
        n = 1 if kind == "decode" else rng.randint(2, 32)
        old = _log(rng, 1, max(2, min(200_000, 4_000_000 // (batch * hk), 400_000_000 // (batch * hq * n))))
    return dict(op=op, batch=batch, n=n, old=old, hq=hq, hk=hk, dim=dim, page=page, dtype=dtype,
                causal=kind == "decode" or rng.random() < 0.6, fresh=kind != "decode" and n * n * batch * hq < 300_000_000
                and rng.random() < 0.5, lse=rng.random() < 0.3, ragged=batch > 1 and rng.random() < 0.6)


def _lengths(most, case):
    """Lengths of the sequences: all the same, or ragged from about most / batch to most, in a fixed shuffled order."""
    b = case["batch"]
    if not case.get("ragged", case["op"] == "write" or case["op"] == "read"):
        return [most] * b
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, b) == 1)
    return [max(1, most * ((i * step) % b + 1) // b) if most else 0 for i in range(b)]


def _plan(case):
    """(query / new rows of each sequence, keys of each sequence already in the cache before the call)."""
    if case["op"] == "read":
        return [0] * case["batch"], _lengths(case["n"], case)
    rows = _lengths(case["n"], case) if case["n"] > 1 else [1] * case["batch"]
    old = _lengths(case["old"], case)[::-1]
    if case["op"] == "attention" and not case["fresh"] and case["causal"]:
        old = [max(o, r) for o, r in zip(old, rows)]  # the queries' own tokens are the last ones in the cache
    return rows, old


# ----------------------------------------------------------------------------------------------------- plain NVFP4
def _quantise(x, g):
    """x [..., D] -> (codes uint8 [..., D / 2], scales uint8 [..., D / 16]), in the order of roundings of the format."""
    g = np.float32(g)
    blocks = x.float().unflatten(-1, (-1, 16))
    wanted = blocks.abs().amax(-1) * float(np.float32(1) / (np.float32(6) * g))
    scale = wanted.clamp(max=448.0).to(torch.float8_e4m3fn)
    step = scale.float() * float(g)
    y = blocks * torch.where(step == 0, 0.0, 1.0 / step)[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8)


def _values(codes, scales, g):
    """The values that codes [..., D / 2] and scales [..., D / 16] stand for, fp32 [..., D]."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return (v.unflatten(-1, (-1, 16)) * scales.view(torch.float8_e4m3fn).float()[..., None] * float(np.float32(g))).flatten(-2)


# ---------------------------------------------------------------------------------------------------------- prepare
def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _cumulative(rows):
    return [0] + np.cumsum(rows).tolist()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + 17)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    if case["op"] == "rope":
        b, n, axes = case["batch"], case["n"], AXES[case["axes"]]
        s = {"case": case, "q": normal(b, n, case["hq"], case["dim"]).to(dtype),
             "k": normal(b, n, case["hk"], case["dim"]).to(dtype), "wq": None, "wk": None}
        if case["norm"]:
            s["wq"], s["wk"] = normal(case["dim"]) * 0.05 + 1, normal(case["dim"]) * 0.05 + 1
        side = max(1, math.isqrt(n))  # a frame number and a centred grid, or text positions deep in a long context
        at = torch.arange(n, device=dev)
        ids = torch.stack([at // (side * side), at // side % side - side // 2, at % side - side // 2], -1)
        ids = ids[:, 3 - len(axes):].expand(b, n, len(axes))
        start = torch.randint(100_000 if case["far"] else 0, 1_000_000 if case["far"] else 300, (b, 1, 1), generator=g, device=dev)
        s["ids"] = (ids + start).float().contiguous()
        return s

    rows, old = _plan(case)
    page, hk, dim, b = case["page"], case["hk"], case["dim"], case["batch"]
    room = [o + (r if case["op"] == "write" else 0) for o, r in zip(old, rows)]
    need = [-(-max(1, r) // page) for r in room]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(b, max(need), dtype=torch.int32, device=dev)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    spread = torch.exp(0.3 * normal(dim))  # some channels of keys run larger than others
    s = {"case": case, "table": table, "k_global": 6.0 / 2688, "v_global": 5.0 / 2688,
         "old": _ints(old, dev), "cu": _ints(_cumulative(rows), dev), "most": (max(rows), max(old))}
    for name, shape in (("k", spread), ("v", torch.ones_like(spread))):
        codes = torch.empty(pages, hk, page, dim // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(pages, hk, page, dim // 16, dtype=torch.uint8, device=dev)
        part = max(1, (1 << 26) // (hk * page * dim))
        for p in range(0, pages, part):
            x = (normal(min(part, pages - p), hk, page, dim) * shape).to(torch.bfloat16)
            codes[p:p + part], scales[p:p + part] = _quantise(x, s[name + "_global"])
        s[name + "_codes"], s[name + "_scales"] = codes, scales
    if case["op"] == "read":
        s["first"], s["cu"] = torch.zeros_like(s["old"]), _ints(_cumulative(old), dev)
        s["total"] = sum(old)
        return s
    if case["op"] == "write":
        s["first"], s["whole_cu"] = torch.zeros_like(s["old"]), _ints(_cumulative(room), dev)
        s["total"], s["most"] = sum(room), (max(rows), max(room))
        # 16-bit rows as they lie in a fused projection's output
        kv = normal(sum(rows), 2, hk, dim)
        kv[:, 0] *= spread
        kv = kv.to(dtype)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        return s
    s["q"] = normal(sum(rows), case["hq"], dim).to(dtype)
    if case["fresh"]:
        s["k"], s["v"] = (normal(sum(rows), hk, dim) * spread).to(dtype), normal(sum(rows), hk, dim).to(dtype)
    return s


# -------------------------------------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    return {"rope": _rope, "write": _write, "read": _read, "attention": _attention}[op](state)


def _rope(s):
    c = s["case"]
    if own:
        kernels, _ = _framework()
        return kernels.rope_axes(s["q"], s["k"], s["ids"], AXES[c["axes"]], 10000.0, wq=s["wq"], wk=s["wk"], eps=1e-6,
                                 interleaved=c["interleaved"], sections=c["sections"], inverse=c["inverse"])
    axes, dev = AXES[c["axes"]], s["q"].device
    half = sum(axes) // 2
    which = torch.repeat_interleave(torch.arange(len(axes), device=dev), torch.tensor([a // 2 for a in axes], device=dev), output_size=half)
    width = torch.tensor([float(sum(axes) if c["sections"] else a) for a in axes], dtype=torch.float64, device=dev)[which]
    first = torch.tensor([0.0 if c["sections"] else float(sum(axes[:i]) // 2) for i in range(len(axes))], dtype=torch.float64, device=dev)[which]
    pair = torch.arange(half, dtype=torch.float64, device=dev) - first
    angle = s["ids"].double()[..., which] * 10000.0 ** (-2 * pair / width)  # 64 bits: far positions
    if c["inverse"]:
        angle = -angle
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    return tuple(_turn(c, s[x], s["w" + x], cos, sin, half) for x in ("q", "k"))


def _turn(c, x, w, cos, sin, half):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
    rot, rest = y[..., :2 * half], y[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if c["interleaved"] else (rot[..., :half], rot[..., half:])
    u, v = cos * a - sin * b, sin * a + cos * b
    rot = torch.stack([u, v], -1).flatten(-2) if c["interleaved"] else torch.cat([u, v], -1)
    return torch.cat([rot, rest], -1).to(x.dtype)


def _cache(s):
    _, kv4 = _framework()
    return kv4.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["k_global"], s["v_global"])


def _places(s, first, cu, total):
    """(page, row in the page) of every row of a packed batch whose sequence b starts at position first[b]."""
    page = s["case"]["page"]
    rows = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu[1:].long(), rows, right=True)
    p = rows - cu.long()[b] + first.long()[b]
    return s["table"].long()[b, p // page], p % page


def _whole(s, cu):
    """All cached rows [0, length) of every sequence, packed, as 16-bit (or 32-bit) values."""
    c, total = s["case"], s["total"]
    dtype = DTYPES[c["dtype"]]
    if own:
        _, kv4 = _framework()
        k = torch.empty(total, c["hk"], c["dim"], dtype=dtype, device=cu.device)
        v = torch.empty_like(k)
        kv4.read(_cache(s), s["table"], s["first"], k, v, cu=cu)
        return k, v
    at = _places(s, s["first"], cu, total)
    return tuple(_values(s[x + "_codes"][at[0], :, at[1]], s[x + "_scales"][at[0], :, at[1]], s[x + "_global"]).to(dtype)
                 for x in ("k", "v"))


def _read(s):
    return _whole(s, s["cu"])


def _write(s):
    if own:
        _, kv4 = _framework()
        kv4.write(_cache(s), s["table"], s["old"], s["k"], s["v"], cu=s["cu"])
    else:
        at = _places(s, s["old"], s["cu"], s["k"].shape[0])
        kc, ks = _quantise(s["k"], s["k_global"])
        vc, vs = _quantise(s["v"], s["v_global"])
        s["k_codes"][at[0], :, at[1]], s["k_scales"][at[0], :, at[1]] = kc, ks
        s["v_codes"][at[0], :, at[1]], s["v_scales"][at[0], :, at[1]] = vc, vs
    return _whole(s, s["whole_cu"])


def _attention(s):
    c = s["case"]
    fresh = c["fresh"]
    if own:
        _, kv4 = _framework()
        return kv4.attention(s["q"], _cache(s), s["table"], s["old"], cu=s["cu"], causal=c["causal"],
                             k_new=s["k"] if fresh else None, v_new=s["v"] if fresh else None, return_lse=c["lse"])
    dev, hk, dim, b = s["q"].device, c["hk"], c["dim"], c["batch"]
    group, (lq, lk) = c["hq"] // hk, s["most"]
    cu, old = s["cu"].long(), s["old"].long()
    rows = cu[1:] - cu[:-1]
    t = torch.arange(s["q"].shape[0], device=dev)
    seq = torch.searchsorted(cu[1:], t, right=True)
    at = t - cu[seq]
    q = torch.zeros(b, lq, c["hq"], dim, device=dev)
    q[seq, at] = s["q"].float()
    q = q.view(b, lq, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(b, hk, group * lq, dim)
    pos = torch.arange(lk, device=dev)
    where = s["table"].long()[:, pos // c["page"]], (pos % c["page"]).expand(b, lk)
    k, v = (_values(s[x + "_codes"][where[0], :, where[1]], s[x + "_scales"][where[0], :, where[1]], s[x + "_global"])
            for x in ("k", "v"))
    inside = pos[None] < old[:, None]  # [b, lk]
    v = v * inside[..., None, None]
    query = torch.arange(lq, device=dev)
    seen = inside[:, None].expand(b, lq, lk)
    if c["causal"] and not fresh:  # the queries are the last rows of the cache
        seen = seen & (pos[None, None] <= (old - rows)[:, None, None] + query[None, :, None])
    if fresh:
        kn, vn = torch.zeros(b, lq, hk, dim, device=dev), torch.zeros(b, lq, hk, dim, device=dev)
        kn[seq, at], vn[seq, at] = s["k"].float(), s["v"].float()
        k, v = torch.cat([k, kn], 1), torch.cat([v, vn], 1)
        new = (query[None, None] < rows[:, None, None]).expand(b, lq, lq)
        if c["causal"]:
            new = new & (query[None, None] <= query[None, :, None])
        seen = torch.cat([seen, new], 2)
    k, v = k.transpose(1, 2), v.transpose(1, 2)  # [b, hk, keys, dim]
    score = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(dim)).view(b, hk, group, lq, -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(b, hk, group * lq, -1) @ v
    out = out.view(b, hk, group, lq, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, lq, c["hq"], dim)[seq, at].to(s["q"].dtype)
    if not c["lse"]:
        return out
    lse = torch.where(total > 0, top + torch.log(total), -math.inf).squeeze(-1)
    return out, lse.permute(0, 3, 1, 2).reshape(b, lq, c["hq"])[seq, at]


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    item = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        n, h = case["batch"] * case["n"], case["hq"] + case["hk"]
        values = n * h * case["dim"]
        return {"bytes": 2 * values * item + n * len(AXES[case["axes"]]) * 4, "flops": values * (7 if case["norm"] else 3)}
    rows, old = _plan(case)
    hk, dim = case["hk"], case["dim"]
    cached = 2 * hk * (dim // 2 + dim // 16)  # bytes of one token's keys and values in the cache
    full = 2 * hk * dim * item
    if case["op"] == "read":
        return {"bytes": sum(old) * (cached + full), "flops": sum(old) * 4 * hk * dim}
    if case["op"] == "write":  # the new rows in and out, then every row in and out
        n, m = sum(rows), sum(rows) + sum(old)
        return {"bytes": n * (full + cached) + m * (cached + full), "flops": n * 6 * hk * dim + m * 4 * hk * dim}
    pairs = 0
    for r, o in zip(rows, old):
        if case["fresh"]:
            pairs += r * o + (r * (r + 1) // 2 if case["causal"] else r * r)
        else:
            pairs += r * o - (r * (r - 1) // 2 if case["causal"] else 0)
    moved = sum(old) * cached + 2 * sum(rows) * case["hq"] * dim * item
    if case["fresh"]:
        moved += sum(rows) * full
    if case["lse"]:
        moved += sum(rows) * case["hq"] * 4
    return {"bytes": moved, "flops": 4 * pairs * case["hq"] * dim}


# ------------------------------------------------------------------------------------------------------------ exact
def _decode64(codes, scales, g):
    """Values of E2M1 codes and E4M3 scales from the bits' meaning, in 64 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    e, m = (n >> 1) & 3, n & 1
    x = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * 2.0 ** (e - 1).double()) * (1 - 2 * (n >> 3)).double()
    t = scales.long()
    e, m = (t >> 3) & 15, t & 7
    f = torch.where(e == 0, m.double() * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7).double()) * (1 - 2 * (t >> 7)).double()
    return x * torch.repeat_interleave(f, 16, -1) * float(np.float32(g))


def _stored64(x, g):
    """The values that x stands for in the cache. The format itself has four steps in 32 bits (the reciprocal of 6 g, a
    block's largest over it, the reciprocal of scale times g, and x times that), which decide which way a value next to a
    border of the 4-bit grid goes: those are rounded here too, all else is in 64 bits."""
    r32 = lambda t: t.float().double()  # noqa: E731
    g = float(np.float32(g))
    blocks = x.double().unflatten(-1, (-1, 16))
    want = r32(blocks.abs().amax(-1) * float(np.float32(1.0 / float(np.float32(6 * g))))).clamp(max=448.0)
    unit = 2.0 ** (torch.floor(torch.log2(want.clamp(min=2.0 ** -6))) - 3)
    step = torch.round(want / unit) * unit * g
    y = r32(blocks * r32(1 / r32(torch.where(step == 0, math.inf, step)))[..., None])
    unit = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return ((torch.round(y / unit) * unit).clamp(-6, 6) * step[..., None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    page, rows = case["page"], (s["cu"][1:] - s["cu"][:-1]).tolist()
    old, cu = s["old"].tolist(), s["cu"].tolist()

    def cached(b, x, n):
        p = torch.arange(n, device=s["table"].device)
        i, r = s["table"][b].long()[p // page], p % page
        return _decode64(s[x + "_codes"][i, :, r], s[x + "_scales"][i, :, r], s[x + "_global"])

    if case["op"] == "read":
        return tuple(torch.cat([cached(b, x, old[b]) for b in range(case["batch"])]) for x in ("k", "v"))
    if case["op"] == "write":
        return tuple(torch.cat([torch.cat([cached(b, x, old[b]), _stored64(s[x][cu[b]:cu[b + 1]], s[x + "_global"])])
                                for b in range(case["batch"])]) for x in ("k", "v"))
    outs, lses = [], []
    group = case["hq"] // case["hk"]
    for b in range(case["batch"]):
        q = s["q"][cu[b]:cu[b + 1]].double()
        k, v = cached(b, "k", old[b]), cached(b, "v", old[b])
        i = torch.arange(rows[b], device=q.device)[:, None]
        last = torch.full_like(i, old[b] - 1)  # the last position that a query sees
        if case["fresh"]:
            k, v = torch.cat([k, s["k"][cu[b]:cu[b + 1]].double()]), torch.cat([v, s["v"][cu[b]:cu[b + 1]].double()])
            last = old[b] + (i if case["causal"] else torch.full_like(i, rows[b] - 1))
        elif case["causal"]:
            last = old[b] - rows[b] + i
        hidden = torch.arange(k.shape[0], device=q.device)[None] > last
        o, e = torch.empty_like(q), torch.empty(rows[b], case["hq"], dtype=torch.float64, device=q.device)
        for h in range(case["hq"]):
            score = (q[:, h] @ k[:, h // group].T / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
            e[:, h] = torch.logsumexp(score, -1)
            o[:, h] = torch.softmax(score, -1).nan_to_num_(0.0) @ v[:, h // group]
        outs.append(o)
        lses.append(e)
    return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)


def _exact_rope(case, s):
    axes, outs = AXES[case["axes"]], []
    half, ids = sum(axes) // 2, s["ids"].double()
    for name in ("q", "k"):
        x = s[name].double()
        if case["norm"]:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s["w" + name].double()
        y, p = x.clone(), 0
        for axis, width in enumerate(axes):
            for i in range(width // 2):
                freq = 10000.0 ** (-2.0 * p / (2 * half)) if case["sections"] else 10000.0 ** (-2.0 * i / width)
                turn = torch.polar(torch.ones_like(ids[..., axis]), ids[..., axis] * freq)[..., None]
                lo, hi = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + half)
                z = torch.complex(x[..., lo], x[..., hi]) * (turn.conj() if case["inverse"] else turn)
                y[..., lo], y[..., hi] = z.real, z.imag
                p += 1
        outs.append(y)
    return tuple(outs)
