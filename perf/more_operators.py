"""What is measured of the paged cache's further operators: the append that rotates queries
and keys on the way into the pages, the same into pages of 4-bit values (with the read that
gives rows back), one-token attention over 4-bit pages, and attention over the pages that a
score selects for each query.

``run`` computes them in elementary torch operations (fp32 or fp64, rounded once), or, where
``own`` is true, by the framework's entry points.  Lengths follow from the case alone
(``_lengths``), values from the seed.

Pages of 4-bit values: uint8 [pages, kv heads, page size * P * 9 / 16] with P the head
dimension rounded up to 64, 128 or 256.  16 slots form a record of 16 * P / 2 bytes of codes
(byte i of a slot: column 2i in the low half, 2i + 1 in the high one; e2m1: sign, then one of
0, 0.5, 1, 1.5, 2, 3, 4, 6) and 16 * P / 16 bytes of scales (e4m3, one for 16 columns).  A
value is code * scale * the cache's own factor.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# up to which magnitude (in units of the scale) a value takes the level; on a border, the level of even index
BORDERS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def _rope(name, dtype, batch, heads, kv_heads, head_dim, rope_dim, page, min_new, max_new, past, bits=0):
    return dict(name=name, op="rope", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                rope_dim=rope_dim, page=page, min_new=min_new, max_new=max_new, past=past, bits=bits)


def _decode4(name, dtype, batch, heads, kv_heads, head_dim, page, min_len, max_len, window=0, sinks=0):
    return dict(name=name, op="decode4", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, min_len=min_len, max_len=max_len, window=window, sinks=sinks)


def _sparse(name, dtype, batch, heads, kv_heads, head_dim, page, min_len, max_len, topk, first, last, max_new=1, bits=0):
    return dict(name=name, op="sparse", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, min_len=min_len, max_len=max_len, topk=topk, first=first, last=last, max_new=max_new, bits=bits)


def listed():
    return [
        # a decode step of the 8-layer model's heads for a batch of requests: one token per row
        _rope("rope_step", "bf16", 32, 8, 2, 128, 128, 64, 1, 1, 767),
        # a batch of long prompts, rotated and put into their pages
        _rope("rope_prompt", "bf16", 8, 32, 8, 128, 128, 16, 1025, 8192, 33),
        # chunks of prompts of an fp32 layer that rotates the first 64 columns of its heads
        _rope("rope_chunk_fp32", "fp32", 24, 8, 2, 128, 64, 32, 3, 257, 1000),
        # a server's step into 4-bit pages, and the rows read back
        _rope("rope4_step", "bf16", 128, 32, 8, 128, 128, 64, 1, 1, 4095, 4),
        # prompts into 4-bit pages and back (what prompt attention of a next chunk reads)
        _rope("rope4_prompt", "fp16", 8, 16, 8, 128, 128, 64, 513, 4096, 77, 4),
        # one user, a short chat over a 4-bit cache: latency
        _decode4("decode4_one_short", "bf16", 1, 8, 2, 128, 64, 517, 517),
        # a server's ragged batch, some rows nearly empty
        _decode4("decode4_batch_8k", "bf16", 32, 32, 8, 128, 64, 1, 8192),
        # few rows over very long caches
        _decode4("decode4_long_128k", "fp16", 4, 32, 8, 128, 16, 100003, 131072),
        # one user with a long context: the latency of scoring, selecting and attending
        _sparse("sparse_one_64k", "bf16", 1, 8, 2, 128, 64, 65001, 65001, 32, 1, 2),
        # a batch over long caches, 1 in 16 pages
        _sparse("sparse_batch_32k", "bf16", 32, 32, 8, 128, 64, 16385, 32768, 32, 1, 2),
        # eight new tokens of each row at once (a draft that is checked), each with pages of its own
        _sparse("sparse_draft_fp16", "fp16", 8, 32, 8, 128, 32, 9000, 16384, 48, 1, 4, 8),
        # 4-bit pages under selection
        _sparse("sparse4_long_128k", "bf16", 4, 32, 8, 128, 64, 100003, 131072, 64, 1, 2, 1, 4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "rope4", "rope4", "decode4", "decode4", "decode4", "sparse", "sparse", "sparse", "sparse4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads, kv = rng.choice([(8, 2), (32, 8), (16, 16), (16, 2), (8, 1), (12, 4), (10, 2)])
    head_dim = rng.choice([128, 128, 64, 96, 80])
    bits = 4 if op.endswith("4") else 0
    page = rng.choice([16, 32, 64, 128, 48])
    room = (8 if dtype == "fp32" else 16) * 8 * 128 * 32768     # cache elements of one of K, V
    if op.startswith("rope"):
        max_new = rng.choice([1, _log_int(rng, 1, 4096)])
        batch = min(_log_int(rng, 1, 128), max(1, 24576 // max_new))
        rope_dim = rng.choice([head_dim, head_dim, head_dim // 2, 32])
        case = _rope("", dtype, batch, heads, kv, head_dim, rope_dim, page, 1 if max_new == 1 else rng.randint(0, max_new),
                     max_new, rng.randint(0, 5000), bits)
    elif op == "decode4":
        max_len = _log_int(rng, 1, 131072)
        batch = min(_log_int(rng, 1, 128), max(1, room // (max_len * kv * head_dim)))
        window = rng.choice([0, 0, 0, _log_int(rng, 1, 8192)])
        case = _decode4("", dtype, batch, heads, kv, head_dim, page, rng.randint(0, max_len), max_len, window,
                        rng.choice([0, 4, 17]) if window else 0)
    else:
        max_len = _log_int(rng, 64, 65536)
        batch = min(_log_int(rng, 1, 64), max(1, room // (2 * max_len * kv * head_dim)))
        topk = rng.randint(2, max(2, min(64, 4096 // page)))
        first = rng.randint(0, 1)
        last = rng.randint(1, topk - first)
        most = max(1, min(128 * 8 * 2048 // (batch * kv * topk * page), 2048 // (batch * kv)))
        case = _sparse("", dtype, batch, heads, kv, head_dim, page, rng.randint(0, max_len), max_len, topk, first,
                       min(last, 4), rng.choice([1, 1, min(most, rng.randint(2, 16))]), bits)
    del case["name"]
    return case


def _lengths(lo, hi, n):
    """n lengths in [lo, hi], spread evenly in a fixed mixed order; the first is hi."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n)]


def _new(c):
    """New tokens of each row, and the slots in use once they are there."""
    if c["op"] == "rope":
        new = _lengths(c["min_new"], c["max_new"], c["batch"])
        return new, [a + b for a, b in zip(new, _lengths(c["past"] // 2, c["past"], c["batch"]))]
    lens = _lengths(c["min_len"], c["max_len"], c["batch"])
    if c["max_new"] == 1:
        return [1] * c["batch"], lens
    return [min(a, n) for a, n in zip(_lengths(1, c["max_new"], c["batch"]), lens)], lens


def _visible(c, n):
    """Visible slots of a row of n."""
    if not c["window"]:
        return n
    lo = max(0, n - c["window"])
    return n - lo + min(c["sinks"], lo)


def work(case):
    c, es = case, 4 if case["dtype"] == "fp32" else 2
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    row4 = D * 9 / 16                                           # bytes of a slot and kv head in 4 bits
    if c["op"] == "rope":
        new, lens = _new(c)
        t = sum(new)
        at = {}
        for n, end in zip(new, lens):
            if n:
                at[end] = max(at.get(end, 0), n)
        # the rows of the tables that are needed: positions of all rows, each once
        spans, rows, top = sorted((end - n, end) for end, n in at.items()), 0, 0
        for lo, hi in spans:
            rows += max(0, hi - max(lo, top))
            top = max(top, hi)
        by = t * (2 * G + H) * D * es + t * H * D * es + rows * c["rope_dim"] * 8 + 12 * c["batch"]
        by += t * 2 * G * (row4 * 2 + D * es if c["bits"] else D * es)
        return {"bytes": by, "flops": 3 * t * (H + G) * c["rope_dim"]}
    if c["op"] == "decode4":
        vis = sum(_visible(c, n) for n in _lengths(c["min_len"], c["max_len"], c["batch"]))
        by = 2 * vis * G * row4 + 2 * c["batch"] * H * D * es + c["batch"] * (H * 4 + 4) + 4 * -(-vis // c["page"])
        return {"bytes": by, "flops": 4 * vis * H * D}
    new, lens = _new(c)
    by = flops = 0
    for n, m in zip(new, lens):
        slots = 0
        for i in range(n):
            pages = -(-(m - n + i + 1) // c["page"])
            slots += min(m - n + i + 1, c["topk"] * c["page"])
            flops += 4 * G * D * pages
        flops += 4 * slots * H * D
        by += 2 * G * min(slots, m) * (row4 if c["bits"] else D * es)
        by += -(-m // c["page"]) * (G * 2 * D * es + 4)
        by += n * (2 * H * D * es + 4 * H + 4 * G * c["topk"])
    return {"bytes": by, "flops": flops}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _padded(dim):
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


def _table(c, cap, gen):
    """Every row's slots in shuffled pages of one pool."""
    width = max(1, -(-cap // c["page"]))
    n = c["batch"] * width + 3
    table = torch.randperm(n, generator=gen, device="cuda")[: c["batch"] * width].view(c["batch"], width).to(torch.int32)
    return table.contiguous(), n


def _pages(c, n, gen, dtype):
    shape = (n, c["page"], c["kv_heads"], c["head_dim"])
    return (torch.randn(shape, generator=gen, device="cuda", dtype=dtype),
            torch.randn(shape, generator=gen, device="cuda", dtype=dtype))


def _pages4(c, n, gen):
    """Pages of 4-bit values as standard normal ones leave them: all codes about equally often, scales near 0.35."""
    P, records = _padded(c["head_dim"]), c["page"] // 16
    both = []
    for _ in range(2):
        x = torch.randint(0, 256, (n, c["kv_heads"], records, 9 * P), generator=gen, device="cuda", dtype=torch.uint8)
        codes = x[..., : 8 * P].view(n, c["kv_heads"], records, 16, P // 2)
        codes[..., (c["head_dim"] + 1) // 2:] = 0
        scales = x[..., 8 * P:]
        scales.remainder_(9).add_(0x28)                          # 0.25 to 0.5
        both.append(x.view(n, c["kv_heads"], records * 9 * P))
    return both


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lengths):
    return _i32([0] + torch.tensor(lengths).cumsum(0).tolist())


def _angles(positions, dim):
    """Tables of the rotation in halves, [positions, dim]: both halves the same angles."""
    f = 1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    a = torch.outer(torch.arange(positions, device="cuda", dtype=torch.float64), f)
    return torch.cat([a.cos(), a.cos()], dim=1).float(), torch.cat([a.sin(), a.sin()], dim=1).float()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    G, H, D = c["kv_heads"], c["heads"], c["head_dim"]
    s = dict(case=c)
    if c["op"] == "rope":
        new, lens = _new(c)
        t, before = sum(new), [m - n for m, n in zip(lens, new)]
        s["table"], n = _table(c, max(lens), gen)
        s["pages_k"], s["pages_v"] = _pages4(c, n, gen) if c["bits"] else _pages(c, n, gen, dt)
        s["lens"], s["after"], s["seen"] = _i32(before), _i32(lens), _i32(before)
        s["new"] = max(new)
        s["cu"] = _cu(new)
        s["each"] = c["min_new"] == c["max_new"] == 1            # one token per row: no offsets needed
        s["cos"], s["sin"] = _angles(max(lens), c["rope_dim"])
        s["q"] = torch.randn(t, H, D, generator=gen, device="cuda", dtype=dt)
        s["k"] = torch.randn(t, G, D, generator=gen, device="cuda", dtype=dt)
        s["v"] = torch.randn(t, G, D, generator=gen, device="cuda", dtype=dt)
        s["q_out"] = torch.zeros_like(s["q"])
        if c["bits"]:
            s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    if c["op"] == "decode4":
        lens, t = _lengths(c["min_len"], c["max_len"], c["batch"]), c["batch"]
        s["table"], n = _table(c, c["max_len"], gen)
        s["pages_k"], s["pages_v"] = _pages4(c, n, gen)
    else:
        new, lens = _new(c)
        t = sum(new)
        s["new"] = max(new)
        s["cu"] = None if c["max_new"] == 1 else _cu(new)
        s["table"], n = _table(c, c["max_len"], gen)
        s["pages_k"], s["pages_v"] = _pages4(c, n, gen) if c["bits"] else _pages(c, n, gen, dt)
        # the bounds of every page, without the newest slots: `run` puts those in
        s["bounds"] = torch.zeros(n, 2, G, D, dtype=dt, device="cuda")
        for b in range(c["batch"]):
            for at in range(0, s["table"].shape[1], 256):
                pages = s["table"][b, at: at + 256].long()
                k = _values4(c, s["pages_k"][pages]).to(dt) if c["bits"] else s["pages_k"][pages]
                s["bounds"][pages] = torch.stack([k.amin(1), k.amax(1)], dim=1)
        s["lens"] = _i32(lens)
        _tail_bounds(s, s["lens"].long() - _i32(new).long())
    s["lens"] = _i32(lens)
    # per-head normalised queries and keys have unit rms; trained norm weights sharpen the scores
    s["q"] = (2.0 * torch.randn(t, H, D, generator=gen, device="cuda")).to(dt)
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(t, H, device="cuda")
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "decode4": _own_decode4, "sparse": _own_sparse}[op](state)
    return {"rope": _plain_rope, "decode4": _plain_decode4, "sparse": _plain_sparse}[op](state)


def _own_rope(s):
    from project_chronos_b200 import ops
    cu = None if s["each"] else s["cu"]
    ops.paged_append_rope(s["k"], s["v"], s["pages_k"], s["pages_v"], s["table"], s["lens"], s["seen"], s["cos"], s["sin"],
                          q=s["q"], q_out=s["q_out"], cu_seqlens=cu)
    if not s["case"]["bits"]:
        return [s["q_out"], s["pages_k"], s["pages_v"]]
    ops.paged_gather(s["pages_k"], s["pages_v"], s["table"], s["after"], s["cu"], s["k_out"], s["v_out"])
    return [s["q_out"], s["k_out"], s["v_out"]]


def _own_decode4(s):
    from project_chronos_b200 import ops
    c = s["case"]
    ops.paged_attn_decode4(s["q"], s["pages_k"], s["pages_v"], s["table"], s["lens"], window=c["window"], sinks=c["sinks"],
                           out=s["out"], lse=s["lse"])
    return [s["out"], s["lse"]]


def _own_sparse(s):
    from project_chronos_b200 import ops
    c = s["case"]
    ops.paged_bounds(s["pages_k"], s["bounds"], s["table"], s["lens"], cu_seqlens=s["cu"])
    pages = ops.paged_select(s["q"], s["bounds"], s["table"], s["lens"], c["page"], c["topk"], first=c["first"],
                             last=c["last"], cu_seqlens=s["cu"])
    ops.paged_attn_sparse(s["q"], s["pages_k"], s["pages_v"], s["table"], s["lens"], pages, cu_seqlens=s["cu"],
                          out=s["out"], lse=s["lse"])
    return [s["bounds"], pages, s["out"], s["lse"]]


def _softmax(scores, seen):
    """Softmax of the scores where `seen`; rows that see nothing are zero. Returns (p, log of the sum)."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    return p, (top + torch.log(total)).squeeze(-1)


def _levels():
    return torch.tensor(LEVELS + [-x for x in LEVELS], device="cuda")


def _values4(c, pages):
    """The values [n, slots, G, D] (fp32) that 4-bit pages [n, G, bytes] stand for."""
    P, n, G = _padded(c["head_dim"]), pages.shape[0], pages.shape[1]
    x = pages.view(n, G, -1, 9 * P)
    b = x[..., : 8 * P].reshape(n, G, -1, 16, P // 2)
    codes = torch.stack([b & 15, b >> 4], dim=-1).view(n, G, -1, 16, P)
    scales = x[..., 8 * P:].contiguous().view(torch.float8_e4m3fn).view(n, G, -1, 16, P // 16).float()
    v = _levels()[codes.int()] * scales.repeat_interleave(16, dim=-1)
    return v.view(n, G, -1, P)[..., : c["head_dim"]].transpose(1, 2)


def _codes4(c, x):
    """4-bit codes and scales of rows x [..., D] in 64 bits: (bytes of codes [..., P / 2], bytes of scales [..., P / 16])."""
    P = _padded(c["head_dim"])
    x = torch.nn.functional.pad(x, (0, P - c["head_dim"]))
    top = x.abs().unflatten(-1, (P // 16, 16)).amax(-1)
    scale = (top / 6).clamp(max=448.0).float().to(torch.float8_e4m3fn)
    units = x.abs() / scale.double().repeat_interleave(16, dim=-1)
    level = torch.zeros_like(units, dtype=torch.int32)
    for i, border in enumerate(BORDERS):
        # level i + 1 from the border on, on the border itself where i + 1 is even
        level += (units >= border) if i % 2 else (units > border)
    code = torch.where(x < 0, level + 8, level)
    code = torch.where(scale.double().repeat_interleave(16, dim=-1) == 0, torch.zeros_like(code), code).unflatten(-1, (P // 2, 2))
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.view(torch.uint8)


def _rotated(x, cos, sin):
    """Rows [T, heads, D] with the first columns rotated in halves; cos, sin [T, dim]."""
    r = cos.shape[1]
    a, b = x[..., : r // 2], x[..., r // 2: r]
    turned = torch.cat([-b, a], dim=-1)
    return torch.cat([x[..., :r] * cos[:, None] + turned * sin[:, None], x[..., r:]], dim=-1)


def _plain_rope(s):
    c = s["case"]
    page, T = c["page"], s["k"].shape[0]
    t = torch.arange(T, device="cuda")
    cu = s["cu"].long()
    b = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[b]
    slot, at = s["lens"].long()[b] + i, s["seen"].long()[b] + i
    where = s["table"].long()[b, slot // page]
    cos, sin = s["cos"][at], s["sin"][at]
    s["q_out"].copy_(_rotated(s["q"].float(), cos, sin))
    if not c["bits"]:
        s["pages_k"][where, slot % page] = _rotated(s["k"].float(), cos, sin).to(s["k"].dtype)
        s["pages_v"][where, slot % page] = s["v"]
        return [s["q_out"], s["pages_k"], s["pages_v"]]
    # next to a border of the codes 32 bits would decide differently
    P, G = _padded(c["head_dim"]), c["kv_heads"]
    rows = [(s["pages_k"], _rotated(s["k"].double(), cos.double(), sin.double())), (s["pages_v"], s["v"].double())]
    for pages, x in rows:
        codes, scales = _codes4(c, x)
        record = pages.view(pages.shape[0], G, page // 16, 9 * P)
        at16 = (where, slice(None), slot % page // 16)
        lines = record[..., : 8 * P].unflatten(-1, (16, P // 2))
        lines[at16 + (slot % 16,)] = codes
        lines = record[..., 8 * P:].unflatten(-1, (16, P // 16))
        lines[at16 + (slot % 16,)] = scales
    # the new rows as they are now in the pages
    for pages, out in ((s["pages_k"], s["k_out"]), (s["pages_v"], s["v_out"])):
        record = pages.view(pages.shape[0], G, page // 16, 9 * P)
        b4 = record[..., : 8 * P].unflatten(-1, (16, P // 2))[where, :, slot % page // 16, slot % 16]
        codes = torch.stack([b4 & 15, b4 >> 4], dim=-1).view(T, G, P)
        scales = record[..., 8 * P:].unflatten(-1, (16, P // 16))[where, :, slot % page // 16, slot % 16]
        scales = scales.contiguous().view(torch.float8_e4m3fn).float().repeat_interleave(16, dim=-1)
        out.copy_((_levels()[codes.int()] * scales)[..., : c["head_dim"]])
    return [s["q_out"], s["k_out"], s["v_out"]]


def _plain_decode4(s):
    c = s["case"]
    B, H, G, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    table = s["table"].long()
    cap = table.shape[1] * c["page"]
    slot, n = torch.arange(cap, device="cuda"), s["lens"].long()[:, None]
    seen = slot < n
    if c["window"]:
        seen = seen & ((slot >= n - c["window"]) | (slot < c["sinks"]))
    k = _values4(c, s["pages_k"][table.view(-1)]).reshape(B, cap, G, D).permute(0, 2, 1, 3)
    v = _values4(c, s["pages_v"][table.view(-1)]).reshape(B, cap, G, D).permute(0, 2, 1, 3)
    scores = torch.matmul(s["q"].view(B, G, H // G, D).float(), k.transpose(2, 3)) / math.sqrt(D)
    p, lse = _softmax(scores, seen[:, None, None, :])
    s["out"].copy_(torch.matmul(p, v).view(B, H, D))
    s["lse"].copy_(lse.reshape(B, H))
    return [s["out"], s["lse"]]


def _rows_of(s):
    """Row and visible slots of every token, [T] each."""
    lens = s["lens"].long()
    if s["cu"] is None:
        return torch.arange(lens.shape[0], device="cuda"), lens
    cu = s["cu"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, lens[b] - (cu[b + 1] - t) + 1


def _keys(s, pages):
    c = s["case"]
    return _values4(c, pages) if c["bits"] else pages.float()


def _tail_bounds(s, upto):
    """Bounds of the pages that the newest tokens lie in, from their slots below `upto` [B]."""
    c, page, lens, table = s["case"], s["case"]["page"], s["lens"].long(), s["table"].long()
    span = -(-s["new"] // page) + 1
    j = torch.div((lens - 1).clamp(min=0), page, rounding_mode="floor")[:, None] - torch.arange(span, device="cuda")
    b, i = ((j >= 0) & (j * page < lens[:, None])).nonzero(as_tuple=True)
    at = j[b, i]
    k = _keys(s, s["pages_k"][table[b, at]])
    used = (at[:, None] * page + torch.arange(page, device="cuda") < upto[b][:, None])[:, :, None, None]
    low = torch.where(used, k, torch.full_like(k, math.inf)).amin(1)
    high = torch.where(used, k, torch.full_like(k, -math.inf)).amax(1)
    s["bounds"][table[b, at]] = torch.stack([low, high], dim=1).to(s["bounds"].dtype)


def _plain_sparse(s):
    c = s["case"]
    H, G, D, page, K = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["topk"]
    lens, table = s["lens"].long(), s["table"].long()
    T, rep = s["q"].shape[0], H // G
    row, n = _rows_of(s)
    _tail_bounds(s, lens)
    # no key of a page scores above its bound: sum_d max(q_d low_d, q_d high_d), summed over a kv head's queries
    q = s["q"].view(T, G, rep, D).double()
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    W = table.shape[1]
    score = torch.empty(T, G, W, dtype=torch.float64, device="cuda")
    step = max(1, 2 ** 27 // (W * G * D))
    for t in range(0, T, step):
        both = s["bounds"][table[row[t: t + step]]].double()        # [t, W, 2, G, D]
        score[t: t + step] = (torch.einsum("tgd,twgd->tgw", up[t: t + step], both[:, :, 1])
                              + torch.einsum("tgd,twgd->tgw", down[t: t + step], both[:, :, 0]))
    w = torch.arange(W, device="cuda")
    pages = -(-n // page)
    always = (w < c["first"]) | (w >= pages[:, None] - c["last"])
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where((w < pages[:, None])[:, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :K]
    order = torch.nn.functional.pad(order, (0, K - order.shape[-1]), value=W)
    chosen = torch.where(torch.arange(K, device="cuda") < pages[:, None, None], order, W).sort(dim=-1).values
    chosen = torch.where(chosen < W, chosen, -1)
    # attention over their slots
    step = max(1, 2 ** 28 // (G * K * page * D))
    slots = torch.arange(page, device="cuda")
    for t in range(0, T, step):
        ids = chosen[t: t + step]
        at = table[row[t: t + step][:, None, None], ids.clamp(min=0)]
        g = torch.arange(G, device="cuda")[:, None]
        if c["bits"]:
            k, v = (_values4(c, x[at, g].flatten(0, 2)[:, None])[:, :, 0].view(*at.shape[:2], -1, D)
                    for x in (s["pages_k"], s["pages_v"]))
        else:
            k, v = (x[at, :, g].flatten(2, 3).float() for x in (s["pages_k"], s["pages_v"]))
        seen = (ids[..., None] >= 0) & (ids[..., None] * page + slots < n[t: t + step, None, None, None])
        x = torch.matmul(s["q"][t: t + step].view(-1, G, rep, D).float(), k.transpose(2, 3)) / math.sqrt(D)
        p, lse = _softmax(x, seen.flatten(2)[:, :, None])
        s["out"][t: t + step] = torch.matmul(p, v).reshape(-1, H, D).to(s["out"].dtype)
        s["lse"][t: t + step] = lse.reshape(-1, H)
    return [s["bounds"], chosen.to(torch.int32), s["out"], s["lse"]]


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits, row by row
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "decode4": _exact_decode4, "sparse": _exact_sparse}[case["op"]](s, s["case"])


def _turn(x, cos, sin):
    y, half = x.clone(), cos.shape[1] // 2
    for lo, sign, other in ((0, -1.0, half), (half, 1.0, 0)):
        here, there = slice(lo, lo + half), slice(other, other + half)
        y[..., here] = x[..., here] * cos[:, None, here] + sign * x[..., there] * sin[:, None, here]
    return y


def _nearest(x):
    """Rows x (fp64, columns a multiple of 16) as 4-bit values stand for them."""
    y = x.unflatten(-1, (-1, 16))
    scale = (y.abs().amax(-1, keepdim=True) / 6).clamp(max=448.0).float().to(torch.float8_e4m3fn).double()
    u = y / torch.where(scale == 0, torch.ones_like(scale), scale)
    grid = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    far = (u.abs()[..., None] - grid).abs()
    near = far.amin(-1, keepdim=True)
    # of two levels as near as each other, the one of even index
    index = torch.where(far == near, torch.arange(8, device="cuda") + 8 * (torch.arange(8, device="cuda") % 2), 99).amin(-1) % 8
    return (torch.sign(u) * grid[index] * scale).flatten(-2)


def _exact_rope(s, c):
    cu, before, seen = s["cu"].tolist(), s["lens"].tolist(), s["seen"].tolist()
    q_out, D = s["q_out"].double(), c["head_dim"]
    if c["bits"]:
        k_out, v_out = s["k_out"].double(), s["v_out"].double()
    else:
        k_out, v_out = s["pages_k"].double(), s["pages_v"].double()
    for b in range(c["batch"]):
        rows = slice(cu[b], cu[b + 1])
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        cos, sin = (x[seen[b]: seen[b] + n].double() for x in (s["cos"], s["sin"]))
        q_out[rows] = _turn(s["q"][rows].double(), cos, sin)
        k, v = _turn(s["k"][rows].double(), cos, sin), s["v"][rows].double()
        if c["bits"]:
            pad = (0, -D % 16)
            k_out[rows] = _nearest(torch.nn.functional.pad(k, pad))[..., :D]
            v_out[rows] = _nearest(torch.nn.functional.pad(v, pad))[..., :D]
        else:
            slot = torch.arange(before[b], before[b] + n, device="cuda")
            to = s["table"][b].long()[slot // c["page"]], slot % c["page"]
            k_out[to], v_out[to] = k, v
    return [q_out, k_out, v_out]


def _row(s, c, pages, b, g, slots):
    """Rows [n, D] in 64 bits that the pages hold in the given slots."""
    page, at = s["table"][b].long()[slots // c["page"]], slots % c["page"]
    if not c["bits"] and c["op"] == "sparse":
        return pages[page, at, g].double()
    P = _padded(c["head_dim"])
    record = pages.view(pages.shape[0], pages.shape[1], -1, 9 * P)[page, g, at // 16]
    col = torch.arange(c["head_dim"], device="cuda")
    line = (at % 16)[:, None]
    code = record.gather(1, line * (P // 2) + col // 2).int() >> (4 * (col % 2)) & 15
    e8 = record.gather(1, 8 * P + line * (P // 16) + col // 16).int()
    scale = torch.where(e8 >= 8, (8 + e8 % 8) * 2.0 ** ((e8 // 8).double() - 10), (e8 % 8) * 2.0 ** -9)
    m = code % 8
    value = torch.where(m >= 2, (2 + m % 2) * 2.0 ** ((m // 2).double() - 2), m * 0.5)
    return torch.where(code >= 8, -value, value) * scale


def _attend(q, k, v):
    x = q.double() @ k.T * k.shape[1] ** -0.5
    lse = torch.logsumexp(x, dim=1)
    return torch.exp(x - lse[:, None]) @ v, lse


def _exact_decode4(s, c):
    H, G = c["heads"], c["kv_heads"]
    out, lse = s["out"].double(), s["lse"].double()
    c = dict(c, bits=4)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            lse[b] = -math.inf
            continue
        slots = torch.arange(n, device="cuda")
        if c["window"]:
            slots = torch.cat([slots[: max(0, min(c["sinks"], n - c["window"]))], slots[max(0, n - c["window"]):]])
        for g in range(G):
            heads = slice(g * H // G, (g + 1) * H // G)
            k, v = (_row(s, c, s[x], b, g, slots) for x in ("pages_k", "pages_v"))
            out[b, heads], lse[b, heads] = _attend(s["q"][b, heads], k, v)
    return [out, lse]


def _exact_sparse(s, c):
    H, G, D, page, K = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["topk"]
    bounds, out, lse = s["bounds"].double(), s["out"].double(), s["lse"].double()
    lens, T = s["lens"].tolist(), s["q"].shape[0]
    cu = list(range(c["batch"] + 1)) if s["cu"] is None else s["cu"].tolist()
    pages = torch.full((T, G, K), -1, dtype=torch.int32, device="cuda")
    for b, m in enumerate(lens):
        for j in range(max(0, (m - (cu[b + 1] - cu[b])) // page), -(-m // page)):
            slots = torch.arange(j * page, min(m, j * page + page), device="cuda")
            for g in range(G):
                k = _row(s, c, s["pages_k"], b, g, slots)
                bounds[s["table"][b, j].long(), 0, g], bounds[s["table"][b, j].long(), 1, g] = k.amin(0), k.amax(0)
        for t in range(cu[b], cu[b + 1]):
            n = m - (cu[b + 1] - 1 - t)
            count = -(-n // page)
            if n <= 0:
                lse[t] = -math.inf
                continue
            at = s["table"][b, :count].long()
            for g in range(G):
                heads = slice(g * H // G, (g + 1) * H // G)
                q = s["q"][t, heads].double()
                low, high = bounds[at, 0, g], bounds[at, 1, g]
                score = torch.maximum(q[:, None] * low, q[:, None] * high).sum((0, 2)).tolist()
                rank = sorted(range(count), key=lambda i: (c["first"] <= i < count - c["last"], -score[i] if c["first"] <= i < count - c["last"] else 0, i))
                ids = sorted(rank[:K])
                pages[t, g, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
                slots = (torch.tensor(ids, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
                slots = slots[slots < n]
                out[t, heads], lse[t, heads] = _attend(s["q"][t, heads], _row(s, c, s["pages_k"], b, g, slots),
                                                       _row(s, c, s["pages_v"], b, g, slots))
    return [bounds, pages, out, lse]
