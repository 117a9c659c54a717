"""What is measured of the paged cache operators: attention of one new token over a paged
key-value cache, prompt attention with a sliding window and first tokens that stay
visible, eviction by accumulated attention weight, and the append that fills the pages.

``run`` computes them in elementary torch operations (fp32, rounded once), or, where
``own`` is true, by the framework's entry points.  Lengths follow from the case alone
(``_lengths``), values from the seed.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def _decode(name, dtype, batch, heads, kv_heads, head_dim, page, min_len, max_len, window=0, sinks=0, track=False):
    return dict(name=name, op="decode", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, min_len=min_len, max_len=max_len, window=window, sinks=sinks, track=track)


def _prompt(name, dtype, batch, heads, kv_heads, head_dim, min_q, max_q, past, window=0, sinks=0, pad=0):
    return dict(name=name, op="prompt", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                min_q=min_q, max_q=max_q, past=past, window=window, sinks=sinks, pad=pad)


def _evict(name, dtype, batch, kv_heads, head_dim, page, min_len, max_len, budget, sinks, recent):
    return dict(name=name, op="evict", dtype=dtype, batch=batch, kv_heads=kv_heads, head_dim=head_dim, page=page,
                min_len=min_len, max_len=max_len, budget=budget, sinks=sinks, recent=recent)


def _append(name, dtype, batch, kv_heads, head_dim, page, min_new, max_new, past, track=False):
    return dict(name=name, op="append", dtype=dtype, batch=batch, kv_heads=kv_heads, head_dim=head_dim, page=page,
                min_new=min_new, max_new=max_new, past=past, track=track)


def listed():
    return [
        # one user, a short chat: the latency of a single token on the 8-layer model's heads
        _decode("decode_one_short", "bf16", 1, 8, 2, 128, 16, 517, 517),
        # a batch of requests of the 8-layer model (a 512-token prompt, up to 256 steps), ragged, some empty rows
        _decode("decode_batch_ragged", "bf16", 32, 8, 2, 128, 64, 0, 768),
        # the fp32 layer with its 2048-token window and four first tokens that stay visible
        _decode("decode_window_sinks_fp32", "fp32", 24, 8, 2, 128, 32, 9, 4095, 2048, 4),
        # a server's batch whose attention weights feed the eviction
        _decode("decode_tracked_8k", "bf16", 16, 32, 8, 128, 16, 4001, 8192, track=True),
        # few rows over very long caches: the split over the length
        _decode("decode_long_128k", "fp16", 4, 32, 8, 128, 64, 100003, 131072),
        # a batch of prompts of the 8-layer model, padding rows behind the last one
        _prompt("prompt_batch_512", "bf16", 32, 8, 2, 128, 257, 512, 0, 2048, 0, pad=37),
        # one long prompt under a window with sinks
        _prompt("prompt_window_8k", "fp16", 1, 32, 8, 128, 8191, 8191, 0, 1024, 4),
        # long prompts in chunks: 2048 new tokens each on up to 6144 cached ones
        _prompt("prompt_chunk_8k", "bf16", 4, 32, 8, 128, 1793, 2048, 6144),
        # every step of a bounded cache: one token over the budget
        _evict("evict_step", "bf16", 32, 2, 128, 64, 2049, 2049, 2048, 4, 256),
        # after a long prompt: the cache cut down to an eighth
        _evict("evict_bulk_32k", "fp16", 8, 8, 128, 16, 20011, 32768, 4096, 4, 512),
        # the step's new tokens into their pages
        _append("append_step", "bf16", 32, 2, 128, 64, 1, 1, 767, track=True),
        # a batch of long prompts into their pages
        _append("append_prompt", "bf16", 8, 8, 128, 16, 1025, 8192, 33),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "evict", "append"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads, kv = rng.choice([(8, 2), (32, 8), (16, 16), (16, 2), (8, 1), (12, 4), (10, 2)])
    head_dim = rng.choice([128, 128, 64, 96, 80])
    page = rng.choice([16, 32, 64, 128, 48])
    room = (8 if dtype == "fp32" else 16) * 8 * 128 * 32768     # cache elements of one of K, V
    if op == "decode":
        max_len = _log_int(rng, 1, 131072)
        batch = min(_log_int(rng, 1, 128), max(1, room // (max_len * kv * head_dim)))
        window = rng.choice([0, 0, _log_int(rng, 1, 8192)])
        case = _decode("", dtype, batch, heads, kv, head_dim, page, rng.randint(0, max_len), max_len, window,
                       rng.choice([0, 4, 17]) if window else 0, rng.random() < 0.3)
    elif op == "prompt":
        most = 1024 if dtype == "fp32" else 4096
        max_q = _log_int(rng, 1, most)
        past = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        batch = _log_int(rng, 1, 32)
        while batch > 1 and (batch * max_q * (max_q + past) * heads > 2 ** 30 * (0.25 if dtype == "fp32" else 2)
                             or batch * (max_q + past) > 32768):
            batch -= 1
        window = rng.choice([0, 0, _log_int(rng, 1, 2048)])
        case = _prompt("", dtype, batch, heads, kv, head_dim, rng.randint(0, max_q), max_q, past, window,
                       rng.choice([0, 4, 17]) if window else 0, rng.choice([0, 5]))
    elif op == "evict":
        max_len = _log_int(rng, 2, 32768)
        batch = min(_log_int(rng, 1, 64), max(1, room // (2 * max_len * kv * head_dim)))
        budget = rng.randint(1, max_len)
        sinks = min(4, budget // 2)
        case = _evict("", dtype, batch, kv, head_dim, page, rng.randint(0, max_len), max_len, budget, sinks,
                      rng.randint(0, min(512, budget - sinks)))
    else:
        max_new = _log_int(rng, 1, 8192)
        batch = min(_log_int(rng, 1, 64), max(1, 65536 // max_new))
        case = _append("", dtype, batch, kv, head_dim, page, rng.randint(0, max_new), max_new, rng.randint(0, 1000),
                       rng.random() < 0.5)
    del case["name"]
    return case


def _lengths(lo, hi, n):
    """n lengths in [lo, hi], spread evenly in a fixed mixed order; the first is hi."""
    return [hi] + [lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(1, n)]


def _visible(c, t):
    """Visible keys of a row at position t."""
    if t < 0:
        return 0
    if not c["window"]:
        return t + 1
    lo = max(0, t + 1 - c["window"])
    return t + 1 - lo + min(c["sinks"], lo)


def _qk_lengths(c):
    lq = _lengths(c["min_q"], c["max_q"], c["batch"])
    past = _lengths(c["past"] // 2, c["past"], c["batch"])
    return lq, [a + b for a, b in zip(lq, past)]


def work(case):
    c, es = case, 4 if case["dtype"] == "fp32" else 2
    if c["op"] == "decode":
        lens = _lengths(c["min_len"], c["max_len"], c["batch"])
        vis = sum(_visible(c, n - 1) for n in lens)
        row = c["kv_heads"] * c["head_dim"] * es
        by = 2 * vis * row + 2 * c["batch"] * c["heads"] * c["head_dim"] * es + c["batch"] * (c["heads"] * 4 + 4)
        by += 4 * -(-vis // c["page"])
        if c["track"]:
            by += 8 * sum(lens) * c["kv_heads"]
        return {"bytes": by, "flops": 4 * vis * c["heads"] * c["head_dim"]}
    if c["op"] == "prompt":
        lq, lk = _qk_lengths(c)
        pairs = sum(_visible(c, k - q + i) for q, k in zip(lq, lk) for i in range(q))
        by = (2 * sum(lq) * c["heads"] + 2 * sum(lk) * c["kv_heads"]) * c["head_dim"] * es + 4 * sum(lq) * c["heads"]
        return {"bytes": by, "flops": 4 * pairs * c["heads"] * c["head_dim"]}
    if c["op"] == "evict":
        by = 0
        for n in _lengths(c["min_len"], c["max_len"], c["batch"]):
            m = min(n, c["budget"])
            far = max(0, n - c["budget"])
            # kept rows lie evenly over the slots but for the recent ones, which all lie at the end
            tail = min(c["recent"], far)
            moved = tail + max(0, m - c["recent"] - c["sinks"]) * max(0, far - c["recent"]) // max(1, n - c["recent"])
            by += c["kv_heads"] * (8 * n + 12 * m + 4 * moved * c["head_dim"] * es) + 8
        return {"bytes": by, "flops": 0}
    new = sum(_lengths(c["min_new"], c["max_new"], c["batch"]))
    return {"bytes": 4 * new * c["kv_heads"] * c["head_dim"] * es + (8 * new * c["kv_heads"] if c["track"] else 0) + 12 * c["batch"],
            "flops": 0}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _pages(c, cap, gen, dtype):
    """Key and value pages with every row's slots in shuffled pages, stale values behind the lengths."""
    width = max(1, -(-cap // c["page"]))
    n = c["batch"] * width + 3
    table = torch.randperm(n, generator=gen, device="cuda")[: c["batch"] * width].view(c["batch"], width).to(torch.int32)
    shape = (n, c["page"], c["kv_heads"], c["head_dim"])
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    return k, v, table.contiguous()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lengths):
    return _i32([0] + torch.tensor(lengths).cumsum(0).tolist())


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(case=c)
    if c["op"] == "decode":
        s["k"], s["v"], s["table"] = _pages(c, c["max_len"], gen, dt)
        s["lens"] = _i32(_lengths(c["min_len"], c["max_len"], c["batch"]))
        # per-head normalised queries and keys have unit rms; trained norm weights sharpen the scores
        s["q"] = (2.0 * torch.randn(c["batch"], c["heads"], c["head_dim"], generator=gen, device="cuda")).to(dt)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(c["batch"], c["heads"], device="cuda")
        if c["track"]:
            cap = s["table"].shape[1] * c["page"]
            s["weights"] = torch.rand(c["batch"], c["kv_heads"], cap, generator=gen, device="cuda")
            s["weights_out"] = torch.zeros_like(s["weights"])
    elif c["op"] == "prompt":
        lq, lk = _qk_lengths(c)
        s["max_q"], s["max_k"] = max(lq), max(lk)
        s["cu_q"], s["cu_k"] = _cu(lq), _cu(lk)
        tq, tk = sum(lq) + c["pad"], sum(lk) + c["pad"]
        s["q"] = (2.0 * torch.randn(tq, c["heads"], c["head_dim"], generator=gen, device="cuda")).to(dt)
        s["k"] = torch.randn(tk, c["kv_heads"], c["head_dim"], generator=gen, device="cuda", dtype=dt)
        s["v"] = torch.randn(tk, c["kv_heads"], c["head_dim"], generator=gen, device="cuda", dtype=dt)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(tq, c["heads"], device="cuda")
    elif c["op"] == "evict":
        lens = _lengths(c["min_len"], c["max_len"], c["batch"])
        s["k"], s["v"], s["table"] = _pages(c, c["max_len"], gen, dt)
        s["lens"], s["seen"] = _i32(lens), _i32([n + 100 for n in lens])
        cap = s["table"].shape[1] * c["page"]
        shape = (c["batch"], c["kv_heads"], cap)
        # summed softmax weights are heavy-tailed; tokens nobody looked at share the value zero
        w = torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda") - 3.0)
        s["weights"] = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.05, torch.zeros_like(w), w)
        # earlier evictions took 100 of the tokens seen: positions ascend with one gap
        slot = torch.arange(cap, device="cuda", dtype=torch.int32).expand(shape)
        gap = torch.randint(1, 50, shape[:2] + (1,), generator=gen, device="cuda", dtype=torch.int32)
        s["positions"] = torch.where(slot < gap, slot, slot + 100).contiguous()
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
    else:
        new = _lengths(c["min_new"], c["max_new"], c["batch"])
        past = _lengths(c["past"] // 2, c["past"], c["batch"])
        s["pages_k"], s["pages_v"], s["table"] = _pages(c, c["max_new"] + c["past"], gen, dt)
        s["lens"], s["seen"] = _i32(past), _i32([n + 7 for n in past])
        s["cu"] = None if c["min_new"] == c["max_new"] == 1 else _cu(new)
        s["k"] = torch.randn(sum(new), c["kv_heads"], c["head_dim"], generator=gen, device="cuda", dtype=dt)
        s["v"] = torch.randn(sum(new), c["kv_heads"], c["head_dim"], generator=gen, device="cuda", dtype=dt)
        s["weights"] = s["positions"] = None
        if c["track"]:
            cap = s["table"].shape[1] * c["page"]
            s["weights"] = torch.rand(c["batch"], c["kv_heads"], cap, generator=gen, device="cuda")
            s["positions"] = torch.zeros(c["batch"], c["kv_heads"], cap, device="cuda", dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"decode": _own_decode, "prompt": _own_prompt, "evict": _own_evict, "append": _own_append}[op](state)
    return {"decode": _plain_decode, "prompt": _plain_prompt, "evict": _plain_evict, "append": _plain_append}[op](state)


def _own_decode(s):
    from project_chronos_b200 import ops
    c = s["case"]
    ops.paged_attn_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], window=c["window"], sinks=c["sinks"],
                          weights=s.get("weights"), weights_out=s.get("weights_out"), out=s["out"], lse=s["lse"])
    return [s["out"], s["lse"]] + ([s["weights_out"]] if c["track"] else [])


def _own_prompt(s):
    from project_chronos_b200 import ops
    c = s["case"]
    ops.window_attention(s["q"], s["k"], s["v"], s["cu_q"], cu_seqlens_k=s["cu_k"], window=c["window"], sinks=c["sinks"],
                         out=s["out"], lse=s["lse"])
    return [s["out"], s["lse"]]


def _own_evict(s):
    from project_chronos_b200 import ops
    c = s["case"]
    r = ops.paged_evict(s["k"], s["v"], s["table"], s["lens"], s["seen"], s["weights"], s["positions"], c["budget"],
                        sinks=c["sinks"], recent=c["recent"], weights_out=s["weights_out"], positions_out=s["positions_out"])
    return [s["k"], s["v"], r["lens"], r["weights"], r["positions"], r["src"]]


def _own_append(s):
    from project_chronos_b200 import ops
    ops.paged_append(s["k"], s["v"], s["pages_k"], s["pages_v"], s["table"], s["lens"], cu_seqlens=s["cu"],
                     seen=s["seen"] if s["weights"] is not None else None, weights=s["weights"], positions=s["positions"])
    return [s["pages_k"], s["pages_v"]] + ([s["weights"], s["positions"]] if s["weights"] is not None else [])


def _softmax(scores, seen):
    """Softmax of the scores where `seen`; rows that see nothing are zero. Returns (p, log of the sum)."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    return p, (top + torch.log(total)).squeeze(-1)


def _plain_decode(s):
    c = s["case"]
    B, H, G, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    table = s["table"].long()
    cap = table.shape[1] * c["page"]
    slot, n = torch.arange(cap, device="cuda"), s["lens"].long()[:, None]
    seen = slot < n
    if c["window"]:
        seen = seen & ((slot >= n - c["window"]) | (slot < c["sinks"]))
    k = s["k"][table].view(B, cap, G, D).permute(0, 2, 1, 3).float()
    v = s["v"][table].view(B, cap, G, D).permute(0, 2, 1, 3).float()
    scores = torch.matmul(s["q"].view(B, G, H // G, D).float(), k.transpose(2, 3)) / math.sqrt(D)
    p, lse = _softmax(scores, seen[:, None, None, :])
    s["out"].copy_(torch.matmul(p, v).view(B, H, D))
    s["lse"].copy_(lse.reshape(B, H))
    if not c["track"]:
        return [s["out"], s["lse"]]
    sums = s["weights"] + p.sum(dim=2)
    s["weights_out"].copy_(torch.where((slot < n)[:, None, :], sums, s["weights_out"]))
    return [s["out"], s["lse"], s["weights_out"]]


def _plain_prompt(s):
    c = s["case"]
    B, H, G, D = c["batch"], c["heads"], c["kv_heads"], c["head_dim"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    i, j = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    in_q, in_k = i < lq[:, None], j < lk[:, None]
    at_q = torch.where(in_q, cu_q[:-1, None] + i, 0)
    at_k = torch.where(in_k, cu_k[:-1, None] + j, 0)
    q = s["q"][at_q].view(B, -1, G, H // G, D).permute(0, 2, 3, 1, 4).float()
    k = s["k"][at_k].permute(0, 2, 1, 3)[:, :, None].float()
    v = s["v"][at_k].permute(0, 2, 1, 3)[:, :, None].float()
    t = (lk - lq)[:, None] + i                                  # [B, Lq]: each row's position
    seen = in_k[:, None, :] & (j <= t[:, :, None])
    if c["window"]:
        seen = seen & ((j > t[:, :, None] - c["window"]) | (j < c["sinks"]))
    p, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D), seen[:, None, None])
    out = torch.matmul(p, v).permute(0, 3, 1, 2, 4).reshape(B, -1, H, D)
    s["out"][at_q[in_q]] = out[in_q].to(s["out"].dtype)
    s["lse"][at_q[in_q]] = lse.permute(0, 3, 1, 2).reshape(B, -1, H)[in_q]
    return [s["out"], s["lse"]]


def _plain_evict(s):
    c = s["case"]
    P, budget = c["page"], c["budget"]
    table, w, pos = s["table"].long(), s["weights"], s["positions"]
    slot = torch.arange(w.shape[2], device="cuda")
    n, seen = s["lens"].long()[:, None, None], s["seen"].long()[:, None, None]
    kept_always = (pos < c["sinks"]) | (pos >= seen - c["recent"])
    key = torch.where(kept_always, torch.full_like(w, math.inf), w)
    key = torch.where(slot < n, key, torch.full_like(w, -1.0))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order).contiguous())
    keep = (slot < n) & (rank < budget)
    far = torch.where(keep & (slot >= budget), slot, w.shape[2]).sort(dim=-1).values[..., :budget]
    low = slot[:budget]
    hole = ~keep[..., :budget] & (low < n)
    src = torch.where(hole, far.gather(-1, hole.cumsum(-1).sub(1).clamp(min=0)), low.expand_as(hole))
    src = torch.where(low < n, src, -1)
    b, g, to = hole.nonzero(as_tuple=True)
    at = src[b, g, to]
    for_k = (table[b, to // P], to % P, g)
    from_k = (table[b, at // P], at % P, g)
    s["k"][for_k] = s["k"][from_k]
    s["v"][for_k] = s["v"][from_k]
    m = src.shape[-1]
    for out, x in ((s["weights_out"], w), (s["positions_out"], pos)):
        out[..., :m] = torch.where(src >= 0, x.gather(-1, src.clamp(min=0)), out[..., :m])
    return [s["k"], s["v"], s["lens"].clamp(max=budget), s["weights_out"], s["positions_out"], src.to(torch.int32)]


def _plain_append(s):
    c = s["case"]
    P, T = c["page"], s["k"].shape[0]
    t = torch.arange(T, device="cuda")
    if s["cu"] is None:
        b, i = t, torch.zeros_like(t)
    else:
        cu = s["cu"].long()
        b = torch.searchsorted(cu[1:], t, right=True)
        i = t - cu[b]
    slot = s["lens"].long()[b] + i
    page = s["table"].long()[b, slot // P]
    s["pages_k"][page, slot % P] = s["k"]
    s["pages_v"][page, slot % P] = s["v"]
    if s["weights"] is None:
        return [s["pages_k"], s["pages_v"]]
    s["weights"][b, :, slot] = 0.0
    s["positions"][b, :, slot] = (s["seen"].long()[b] + i).to(torch.int32)[:, None].expand(-1, c["kv_heads"])
    return [s["pages_k"], s["pages_v"], s["weights"], s["positions"]]


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits, row by row
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "decode":
        return _exact_decode(s, c)
    if c["op"] == "prompt":
        return _exact_prompt(s, c)
    if c["op"] == "evict":
        return _exact_evict(s, c)
    return None                     # copies: nothing is computed


def _exact_decode(s, c):
    H, G, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    out = s["out"].double()
    lse = s["lse"].double()
    sums = s["weights_out"].double() if c["track"] else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            lse[b] = -math.inf
            continue
        slots = torch.arange(n, device="cuda")
        if c["window"]:
            slots = torch.cat([slots[: max(0, min(c["sinks"], n - c["window"]))], slots[max(0, n - c["window"]):]])
        rows = s["table"][b].long()[slots // P], slots % P
        for g in range(G):
            heads = slice(g * H // G, (g + 1) * H // G)
            k, v = s["k"][rows[0], rows[1], g].double(), s["v"][rows[0], rows[1], g].double()
            x = s["q"][b, heads].double() @ k.T * D ** -0.5
            lse[b, heads] = torch.logsumexp(x, dim=1)
            p = torch.exp(x - lse[b, heads, None])
            out[b, heads] = p @ v
            if c["track"]:
                sums[b, g, :n] = s["weights"][b, g, :n].double()
                sums[b, g, slots] += p.sum(0)
    return [out, lse] + ([sums] if c["track"] else [])


def _exact_prompt(s, c):
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    out, lse = s["out"].double(), s["lse"].double()
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(c["batch"]):
        nq, nk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        if nq == 0:
            continue
        pos = torch.arange(nk - nq, nk, device="cuda")[:, None]
        key = torch.arange(nk, device="cuda")[None]
        hidden = key > pos
        if c["window"]:
            hidden |= (pos - key >= c["window"]) & (key >= c["sinks"])
        for h in range(H):
            g = h * G // H
            x = (s["q"][cq[b]: cq[b + 1], h].double() @ s["k"][ck[b]: ck[b + 1], g].double().T) * D ** -0.5
            x.masked_fill_(hidden, -math.inf)
            lse[cq[b]: cq[b + 1], h] = torch.logsumexp(x, dim=1)
            out[cq[b]: cq[b + 1], h] = torch.softmax(x, dim=1) @ s["v"][ck[b]: ck[b + 1], g].double()
    return [out, lse]


def _exact_evict(s, c):
    budget = c["budget"]
    w_out, p_out = s["weights_out"].cpu(), s["positions_out"].cpu()
    w_in, p_in = s["weights"].cpu(), s["positions"].cpu()
    src = torch.full((c["batch"], c["kv_heads"], budget), -1, dtype=torch.int32)
    lens, seen = s["lens"].tolist(), s["seen"].tolist()
    for b, n in enumerate(lens):
        m = min(n, budget)
        for g in range(c["kv_heads"]):
            w, p = w_in[b, g, :n].tolist(), p_in[b, g, :n].tolist()
            always = [x < c["sinks"] or x >= seen[b] - c["recent"] for x in p]
            best = sorted(range(n), key=lambda i: (not always[i], 0.0 if always[i] else -w[i], i))[:m]
            kept = set(best)
            movers = iter(sorted(i for i in kept if i >= budget))
            src[b, g, :m] = torch.tensor([i if i in kept else next(movers) for i in range(m)], dtype=torch.int32)
    at = src.long().clamp(min=0)
    w_out[..., :budget] = torch.where(src >= 0, w_in.gather(-1, at), w_out[..., :budget])
    p_out[..., :budget] = torch.where(src >= 0, p_in.gather(-1, at), p_out[..., :budget])
    return [None, None, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), w_out.double(), p_out, src]
