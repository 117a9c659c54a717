"""The paged key-value cache (include/chronos_paged.h): append, one-token attention,
eviction by attention weight, and prompt attention with a window and first tokens.

CPU: refusals of the torch-facing calls and of the C ABI.  GPU: every operator
against its definition in 64 bits.  Tolerances follow from the arithmetic, with
u = finfo(type).eps / 2 and A = sum_j p_j |v_j|:

* a score is a sum of D products accumulated in fp32 (each addition off by at most
  2^-23 of the running sum of magnitudes, also where the tensor core cuts instead of
  rounding), so it is off by at most D 2^-23 S, S = max_j scale sum_d |q_d k_jd|; the
  exponential adds 2^-21 of its value; a weight p_j is thus off by
  f = D 2^-23 S + n 2^-24 + 2^-20 of itself (n: terms of its normalising sum);
* fp32 layers of the tensor-core path split every operand into two tf32 terms: a product is
  off by 2^-21 of its magnitude, which D 2^-23 S (D >= 8 here) and the 2^-20 of f cover
  beside their fewer additions;
* 16-bit layers round the weights to the layer type before the second product (u A) and
  the result once (u |out|); the second product adds n 2^-23 A.
  So |error| <= u (A + |out|) + (f + n 2^-23) A, without the first u A for fp32;
* lse is off by at most f + 2^-22 |lse|; a slot's summed weight by f sum p + rounding.
"""
import ctypes
import math

import pytest
import torch

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def _unit(dt):
    return torch.finfo(dt).eps / 2


# ---------------------------------------------------------------------------------------
# refusals (no GPU)
# ---------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    from project_chronos_b200 import _native, build
    build.build()
    return _native.load_library()


def _cpu_cache(b=2, g=2, d=16, pages=4, size=4, width=2, dt=FP):
    return (torch.zeros(pages, size, g, d, dtype=dt), torch.zeros(pages, size, g, d, dtype=dt),
            torch.zeros(b, width, dtype=torch.int32), torch.ones(b, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    from project_chronos_b200 import ops
    kp, vp, table, lens = _cpu_cache()
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attn_decode(torch.zeros(2, 4, 16), kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_append(torch.zeros(2, 2, 16), torch.zeros(2, 2, 16), kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_evict(kp, vp, table, lens, lens, torch.zeros(2, 2, 8), torch.zeros(2, 2, 8, dtype=torch.int32), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.window_attention(torch.zeros(3, 4, 16), torch.zeros(3, 2, 16), torch.zeros(3, 2, 16),
                             torch.tensor([0, 3], dtype=torch.int32))


def _native_cache(N, **kw):
    f = dict(batch=2, kv_heads=2, head_dim=16, dtype=N.DTYPE_BF16, num_pages=4, page_size=4, table_width=2)
    f.update(kw)
    return N.ChronosPagedCache(**f)


@pytest.mark.parametrize("change, text", [
    (dict(cache=dict(head_dim=0)), b"head_dim"), (dict(cache=dict(head_dim=257)), b"head_dim"),
    (dict(cache=dict(page_size=0)), b"page_size"), (dict(cache=dict(dtype=7)), b"dtype"),
    (dict(cache=dict(batch=-1)), b"batch"), (dict(heads=3), b"heads"), (dict(heads=0), b"heads"),
    (dict(heads=2 * 257), b"heads"), (dict(window=-1), b"window"), (dict(sinks=-1), b"sinks"),
    (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(weights=256), b"weights_out"), ({}, b"required"),
])
def test_decode_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(heads=4, window=0, sinks=0, scale=0.25)
    f.update({k: v for k, v in change.items() if k != "cache"})
    a = N.ChronosPagedDecodeArgs(cache=_native_cache(N, **change.get("cache", {})), **f)
    assert lib.chronos_paged_decode(ctypes.byref(a), None) == N.CHRONOS_ERR_INVALID_ARG
    assert text in lib.chronos_moe_last_error()
    if change:
        assert lib.chronos_paged_decode_workspace(ctypes.byref(a)) == 0


@pytest.mark.parametrize("f, text", [
    (dict(budget=0), b"budget"), (dict(budget=4, sinks=3, recent=2), b"budget"), (dict(budget=4, sinks=-1), b"budget"),
    (dict(budget=4, recent=-1), b"budget"), (dict(budget=4, slot_cap=-1), b"slot_cap"), (dict(budget=4), b"required"),
])
def test_evict_refuses_before_touching_the_device(lib, f, text):
    from project_chronos_b200 import _native as N
    a = N.ChronosPagedEvictArgs(cache=_native_cache(N), **f)
    assert lib.chronos_paged_evict(ctypes.byref(a), None) == N.CHRONOS_ERR_INVALID_ARG
    assert text in lib.chronos_moe_last_error()


@pytest.mark.parametrize("f, text", [
    (dict(num_tokens=-1), b"num_tokens"), (dict(num_tokens=3), b"cu_seqlens"),
    (dict(num_tokens=2, positions=256), b"seen"), (dict(num_tokens=2, weights=256, slot_cap=-1), b"slot_cap"),
    (dict(num_tokens=2), b"required"),
])
def test_append_refuses_before_touching_the_device(lib, f, text):
    from project_chronos_b200 import _native as N
    a = N.ChronosPagedAppendArgs(cache=_native_cache(N), **f)
    assert lib.chronos_paged_append(ctypes.byref(a), None) == N.CHRONOS_ERR_INVALID_ARG
    assert text in lib.chronos_moe_last_error()


@pytest.mark.parametrize("change, text", [
    (dict(heads=3), b"heads"), (dict(kv_heads=0), b"kv_heads"), (dict(head_dim=300), b"head_dim"),
    (dict(dtype=-1), b"dtype"), (dict(window=-2), b"window"), (dict(scale=-1.0), b"scale"),
    (dict(num_q=-1), b"query rows"), (dict(num_k=1 << 31), b"key rows"), ({}, b"required"),
])
def test_window_attention_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(batch=1, heads=4, kv_heads=2, head_dim=16, dtype=N.DTYPE_BF16, scale=0.25, num_q=4, num_k=4)
    f.update(change)
    a = N.ChronosWindowAttnArgs(**f)
    assert lib.chronos_window_attention(ctypes.byref(a), None) == N.CHRONOS_ERR_INVALID_ARG
    assert text in lib.chronos_moe_last_error()


def test_empty_calls_return_without_a_device(lib):
    from project_chronos_b200 import _native as N
    d = N.ChronosPagedDecodeArgs(cache=_native_cache(N, batch=0), heads=4, scale=1.0)
    assert lib.chronos_paged_decode(ctypes.byref(d), None) == N.CHRONOS_OK
    e = N.ChronosPagedEvictArgs(cache=_native_cache(N, batch=0), budget=1)
    assert lib.chronos_paged_evict(ctypes.byref(e), None) == N.CHRONOS_OK
    p = N.ChronosPagedAppendArgs(cache=_native_cache(N, batch=0))
    assert lib.chronos_paged_append(ctypes.byref(p), None) == N.CHRONOS_OK
    w = N.ChronosWindowAttnArgs(batch=0, heads=2, kv_heads=2, head_dim=8, scale=1.0)
    assert lib.chronos_window_attention(ctypes.byref(w), None) == N.CHRONOS_OK


def test_page_bookkeeping_on_the_host():
    from project_chronos_b200 import PagedCache
    c = PagedCache(2, 5, 1, 8, 4, "cpu", torch.float32, page_size=4)
    c.reserve(0, 9)
    c.reserve(1, 1)
    assert c.page_table.tolist() == [[0, 1, 2, -1], [3, -1, -1, -1]] and c.free_pages() == 1
    c.reserve(0, 12)                                     # covered already
    with pytest.raises(RuntimeError, match="at most 4"):
        c.reserve(0, 17)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.reserve(1, 12)
    assert c.page_table.tolist()[1] == [3, -1, -1, -1] and c.free_pages() == 1   # nothing half done
    c.trim(0, 5)
    assert c.page_table.tolist()[0] == [0, 1, -1, -1] and c.free_pages() == 2
    c.reserve(1, 12)
    assert sorted(c.page_table[1, :3].tolist()) == [2, 3, 4]
    c.lens[1] = 12
    c.release(1)
    assert c.page_table.tolist()[1] == [-1] * 4 and c.free_pages() == 3 and c.lens.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(3)
    with pytest.raises(ValueError):
        PagedCache(0, 5, 1, 8, 4, "cpu")


# ---------------------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------------------

def _attend(q, k, v, scale, seen):
    """q [H, D], k and v [n, G, D], seen [n] (or [H, n]): out, lse, p [H, n], and what the
    tolerance needs: A [H, D], f."""
    h, g = q.shape[0], k.shape[1]
    k = k.double().repeat_interleave(h // g, dim=1)
    v = v.double().repeat_interleave(h // g, dim=1)
    seen = seen.expand(h, -1)
    q = q.double()
    x = torch.einsum("hd,nhd->hn", q, torch.where(seen.T[..., None], k, 0.0)) * scale
    x = x.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, dim=1)
    p = torch.where(seen, torch.exp(x - lse[:, None]), 0.0)
    v = torch.where(seen.T[..., None], v, 0.0)
    out = torch.einsum("hn,nhd->hd", p, v)
    a = torch.einsum("hn,nhd->hd", p, v.abs())
    s = (torch.einsum("hd,nhd->hn", q.abs(), torch.where(seen.T[..., None], k, 0.0).abs()) * scale).amax(dim=1) \
        if k.shape[0] else torch.zeros(h, dtype=torch.float64, device=q.device)
    n = k.shape[0]
    f = q.shape[1] * 2.0 ** -23 * s + n * 2.0 ** -24 + 2.0 ** -20
    return out, lse, p, a, f


def _check_out(got, out, a, f, n, dt):
    u = _unit(dt)
    tol = u * out.abs() + (f[:, None] + n * 2.0 ** -23) * a + (u * a if dt != FP else 0.0) + 1e-30
    if dt == HF:
        # below fp16's normal range the result and each of the n weights (relative to a sum of at least 1)
        # step by 2^-24; the values are standard normal, below 6
        tol = tol + 2.0 ** -25 * (1 + 6 * n)
    err = (got.double() - out).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the tolerance"


def _check_lse(got, lse, f):
    none = lse == -math.inf
    assert bool((got.double()[none] == -math.inf).all())
    err = (got.double() - lse).abs()[~none]
    assert bool((err <= (f + 2.0 ** -22 * lse.abs())[~none]).all())


def _visible(n, window, sinks, dev, at=None):
    """Slots a query at the last position (or at position `at`) sees of n."""
    t = n - 1 if at is None else at
    j = torch.arange(n, device=dev)
    seen = j <= t
    if window:
        seen = seen & ((j > t - window) | (j < sinks))
    return seen


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _make_cache(lens, g, d, size, dt, seed, width=None, bad=float("nan")):
    """Shuffled pages; what no sequence owns is `bad`."""
    gen = _gen(seed)
    width = width or max(1, -(-max(lens) // size)) + 1
    b = len(lens)
    pages = b * width + 2
    table = torch.randperm(pages, generator=gen, device="cuda")[: b * width].view(b, width).to(torch.int32)
    kp = torch.full((pages, size, g, d), bad, dtype=dt, device="cuda")
    vp = torch.full((pages, size, g, d), bad, dtype=dt, device="cuda")
    rows = []
    for i, n in enumerate(lens):
        k = torch.randn(n, g, d, generator=gen, device="cuda").to(dt)
        v = torch.randn(n, g, d, generator=gen, device="cuda").to(dt)
        s = torch.arange(n, device="cuda")
        kp[table[i].long()[s // size], s % size] = k
        vp[table[i].long()[s // size], s % size] = v
        rows.append((k, v))
    return kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), rows


# ---------------------------------------------------------------------------------------
# one-token attention
# ---------------------------------------------------------------------------------------

LENS = [0, 1, 15, 16, 17, 63, 64, 65, 333, 1100]


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d, size", [(8, 2, 128, 16), (4, 4, 64, 64), (10, 2, 80, 48), (9, 1, 96, 16), (17, 1, 128, 32),
                                           (16, 2, 256, 16), (6, 3, 40, 7), (2, 1, 37, 5), (3, 3, 1, 1), (40, 1, 8, 16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 0), (64, 4), (7, 100)])
def test_decode_matches_its_definition(dt, h, g, d, size, window, sinks):
    from project_chronos_b200 import ops
    kp, vp, table, lens, rows = _make_cache(LENS, g, d, size, dt, seed=h * d + size)
    q = (2 * torch.randn(len(LENS), h, d, generator=_gen(3), device="cuda")).to(dt)
    lse = torch.full((len(LENS), h), 7.0, device="cuda")
    out = ops.paged_attn_decode(q, kp, vp, table, lens, window=window, sinks=sinks, lse=lse)
    ops.check_status(out.device)
    for b, (k, v) in enumerate(rows):
        n = LENS[b]
        ref, rl, _, a, f = _attend(q[b], k, v, d ** -0.5, _visible(n, window, sinks, "cuda"))
        _check_out(out[b], ref, a, f, n, dt)
        _check_lse(lse[b], rl, f)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h, g, lens", [(8, 1, [20011]), (4, 2, [1, 9000, 3, 0, 5000]), (24, 1, [7001, 64])])
def test_decode_split_over_the_length(dt, h, g, lens):
    from project_chronos_b200 import ops
    d, size = 128, 16
    kp, vp, table, ln, rows = _make_cache(lens, g, d, size, dt, seed=5)
    q = (3 * torch.randn(len(lens), h, d, generator=_gen(6), device="cuda")).to(dt)
    lse = torch.empty(len(lens), h, device="cuda")
    out = ops.paged_attn_decode(q, kp, vp, table, ln, lse=lse)
    again = ops.paged_attn_decode(q, kp, vp, table, ln)
    assert torch.equal(out, again)
    for b, (k, v) in enumerate(rows):
        n = lens[b]
        ref, rl, _, a, f = _attend(q[b], k, v, d ** -0.5, _visible(n, 0, 0, "cuda"))
        _check_out(out[b], ref, a, f, n, dt)
        _check_lse(lse[b], rl, f)


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d, window, sinks", [(8, 2, 128, 0, 0), (20, 2, 64, 100, 3), (6, 6, 36, 0, 0)])
@pytest.mark.parametrize("in_place", [True, False])
def test_decode_adds_attention_weights(dt, h, g, d, window, sinks, in_place):
    from project_chronos_b200 import ops
    lens = [0, 1, 70, 2500, 130]
    kp, vp, table, ln, rows = _make_cache(lens, g, d, 16, dt, seed=8)
    cap = table.shape[1] * 16 + (0 if in_place else 3)
    q = (2 * torch.randn(len(lens), h, d, generator=_gen(9), device="cuda")).to(dt)
    w = torch.rand(len(lens), g, cap, generator=_gen(10), device="cuda")
    before = w.clone()
    to = w if in_place else torch.full_like(w, -5.0)
    out = ops.paged_attn_decode(q, kp, vp, table, ln, window=window, sinks=sinks, weights=w,
                                weights_out=None if in_place else to)
    for b, (k, v) in enumerate(rows):
        n = lens[b]
        ref, _, p, a, f = _attend(q[b], k, v, d ** -0.5, _visible(n, window, sinks, "cuda"))
        _check_out(out[b], ref, a, f, n, dt)
        rep = h // g
        add = p.view(g, rep, n).sum(1)
        want = before[b, :, :n].double() + add
        tol = f.view(g, rep).amax(1)[:, None] * add + (rep + 1) * 2.0 ** -24 * want
        assert bool(((to[b, :, :n].double() - want).abs() <= tol).all())
        behind = before[b, :, n:] if in_place else torch.full_like(before[b, :, n:], -5.0)
        assert torch.equal(to[b, :, n:], behind)
    if not in_place:
        assert torch.equal(w, before)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("layout", ["interleaved", "heads first", "odd strides"])
def test_decode_takes_strides(dt, layout):
    from project_chronos_b200 import ops
    lens, h, g, d, size = [33, 200, 5], 8, 2, 64, 16
    kp, vp, table, ln, rows = _make_cache(lens, g, d, size, dt, seed=21)
    if layout == "interleaved":
        both = torch.stack([kp, vp], dim=1)
        kp, vp = both[:, 0], both[:, 1]
    elif layout == "heads first":
        kp, vp = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (kp, vp))
    else:   # rows of d + 1 elements: no 16-byte copies
        kp, vp = (torch.cat([x, x[..., :1]], dim=-1)[..., :d] for x in (kp, vp))
    fused = (2 * torch.randn(len(lens), h + 2 * g + 1, d, generator=_gen(4), device="cuda")).to(dt)
    wide = torch.full((len(lens), h + 1, d + 2), 9.0, dtype=dt, device="cuda")
    out = wide[:, :h, :d]
    tall = torch.cat([table, table], dim=1)[:, : table.shape[1]]
    ops.paged_attn_decode(fused[:, :h], kp, vp, tall, ln, out=out)
    for b, (k, v) in enumerate(rows):
        ref, _, _, a, f = _attend(fused[b, :h], k, v, d ** -0.5, _visible(lens[b], 0, 0, "cuda"))
        _check_out(out[b], ref, a, f, lens[b], dt)
    assert bool((wide[:, h:] == 9.0).all()) and bool((wide[..., d:] == 9.0).all())


@gpu
def test_decode_offsets_pass_32_bits():
    from project_chronos_b200 import ops
    g, d, size = 8, 128, 64
    pages = (1 << 31) // (g * d * size) + 40      # elements of one of K, V beyond 2^31
    kp = torch.empty(pages, size, g, d, dtype=BF, device="cuda")
    vp = torch.empty(pages, size, g, d, dtype=BF, device="cuda")
    table = torch.tensor([[pages - 1, 2, pages - 7]], dtype=torch.int32, device="cuda")
    n = 150
    k, v = torch.randn(n, g, d, device="cuda").to(BF), torch.randn(n, g, d, device="cuda").to(BF)
    lens = torch.tensor([0], dtype=torch.int32, device="cuda")
    ops.paged_append(k, v, kp, vp, table, lens, cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    s = torch.arange(n, device="cuda")
    assert torch.equal(kp[table[0].long()[s // size], s % size], k)
    q = torch.randn(1, 16, d, device="cuda").to(BF)
    lens.fill_(n)
    out = ops.paged_attn_decode(q, kp, vp, table, lens)
    ref, _, _, a, f = _attend(q[0], k, v, d ** -0.5, _visible(n, 0, 0, "cuda"))
    _check_out(out[0], ref, a, f, n, BF)
    cap = 3 * size
    r = ops.paged_evict(kp, vp, table, lens, lens, torch.rand(1, g, cap, device="cuda"),
                        torch.arange(cap, dtype=torch.int32, device="cuda").expand(1, g, cap).contiguous(), 70)
    for j in range(g):
        src = r["src"][0, j].long()
        assert torch.equal(kp[table[0].long()[s[:70] // size], s[:70] % size, j], k[src, j])


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_bad_pages_and_lengths_are_reported_and_stay_in_bounds(dt):
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    lens, h, g, d = [40, 100], 4, 2, 64
    kp, vp, table, ln, rows = _make_cache(lens, g, d, 16, dt, seed=2)
    q = torch.randn(2, h, d, device="cuda").to(dt)
    dev = q.device
    ref, _, _, a, f = _attend(q[0], *rows[0], d ** -0.5, _visible(40, 0, 0, "cuda"))
    for page in (-1, kp.shape[0], 1 << 30):
        t = table.clone()
        t[1, 2] = page                            # slots 32..47 of sequence 1 lie nowhere
        w = torch.zeros(2, g, 128, device="cuda")
        out = ops.paged_attn_decode(q, kp, vp, t, ln, weights=w)
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(dev)
        _check_out(out[0], ref, a, f, 40, dt)
        seen = _visible(100, 0, 0, "cuda")
        seen[32:48] = False
        r1, _, p1, a1, f1 = _attend(q[1], *rows[1], d ** -0.5, seen)
        _check_out(out[1], r1, a1, f1, 100, dt)
        assert bool((w[1, :, 32:48] == 0).all()) and bool(torch.isfinite(w).all())
        ops.paged_append(q[:, :g].contiguous(), q[:, :g].contiguous(), kp, vp, t,
                         torch.tensor([60, 33], dtype=torch.int32, device="cuda"))
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(dev)
    for n in (-3, 16 * table.shape[1] + 1, 1 << 30):
        bad = torch.tensor([40, n], dtype=torch.int32, device="cuda")
        out = ops.paged_attn_decode(q, kp, vp, table, bad)
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(dev)
        _check_out(out[0], ref, a, f, 40, dt)
        ops.paged_append(q[:, :g].contiguous(), q[:, :g].contiguous(), kp, vp, table,
                         torch.tensor([50, n], dtype=torch.int32, device="cuda"))
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(dev)
    ops.check_status(dev)


@gpu
def test_decode_refuses_wrong_tensors():
    from project_chronos_b200 import ops
    kp, vp, table, ln, _ = _make_cache([5, 6], 2, 64, 16, BF, seed=1)
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    ok = dict(q=q, k_pages=kp, v_pages=vp, page_table=table, lens=ln)
    for change in (dict(q=q.float()), dict(q=q[:1]), dict(q=q[..., :32]), dict(v_pages=vp.half()), dict(v_pages=vp[:2]),
                   dict(page_table=table.long()), dict(lens=ln.long()), dict(lens=ln[:1]), dict(q=q.cpu()),
                   dict(out=torch.zeros(2, 4, 32, dtype=BF, device="cuda")), dict(lse=torch.zeros(2, 5, device="cuda")),
                   dict(out=torch.zeros(2, 1, 64, dtype=BF, device="cuda").expand(2, 4, 64)),
                   dict(weights=torch.zeros(2, 3, 32, device="cuda")), dict(weights_out=torch.zeros(2, 2, 32, device="cuda")),
                   dict(k_pages=kp.transpose(2, 3).contiguous().transpose(2, 3)), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((TypeError, ValueError)):
            ops.paged_attn_decode(**{**ok, **change})
    with pytest.raises(RuntimeError, match="heads"):
        ops.paged_attn_decode(**{**ok, "q": q[:, :3]})
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.paged_attn_decode(**{**ok, "q": q.clone().requires_grad_()})
    with pytest.raises(ValueError, match="expanded"):
        ops.paged_append(q[:, :2].contiguous(), q[:, :2].contiguous(), kp[:1].expand(4, -1, -1, -1),
                         vp[:1].expand(4, -1, -1, -1), table, ln)


@gpu
def test_decode_graphs_keep_their_own_workspaces():
    """Two captured calls replay at once on two streams while lengths grow."""
    from project_chronos_b200 import ops
    dt, h, g, d = BF, 8, 1, 128
    state = []
    for seed in (1, 2):
        kp, vp, table, ln, rows = _make_cache([6000], g, d, 16, dt, seed=seed)
        q = torch.randn(1, h, d, generator=_gen(seed), device="cuda").to(dt)
        out = torch.empty_like(q)
        w = torch.zeros(1, g, table.shape[1] * 16, device="cuda")
        ln.fill_(100)
        ops.paged_attn_decode(q, kp, vp, table, ln, weights=w, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attn_decode(q, kp, vp, table, ln, weights=w, out=out)
        state.append((kp, vp, table, ln, rows, q, out, w, graph))
    streams = [torch.cuda.Stream() for _ in state]
    for n in (101, 3000, 6000):
        for s in state:
            s[3].fill_(n)
            s[7].zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for st, s in zip(streams, state):
                with torch.cuda.stream(st):
                    s[7].zero_()
                    s[8].replay()
        torch.cuda.synchronize()
        for kp, vp, table, ln, rows, q, out, w, _ in state:
            k, v = rows[0]
            ref, _, p, a, f = _attend(q[0], k[:n], v[:n], d ** -0.5, _visible(n, 0, 0, "cuda"))
            _check_out(out[0], ref, a, f, n, dt)
            assert bool(((w[0, 0, :n].double() - p.sum(0)).abs() <= f.max() * p.sum(0) + h * 2.0 ** -23 * p.sum(0)).all())


# ---------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("g, d, size", [(2, 128, 16), (3, 37, 5), (1, 8, 64), (16, 80, 48)])
@pytest.mark.parametrize("new", [None, [3, 0, 40, 1, 0, 129], [0, 0, 0, 0, 0, 0]])
def test_append_writes_exactly_its_slots(dt, g, d, size, new):
    from project_chronos_b200 import ops
    past = [0, 4, 17, 100, 31, 2]
    b = len(past)
    counts = new or [1] * b
    kp, vp, table, _, _ = _make_cache([p + c for p, c in zip(past, counts)], g, d, size, dt, seed=d, bad=-3.0)
    lens = torch.tensor(past, dtype=torch.int32, device="cuda")
    seen = lens + 1000
    cap = table.shape[1] * size + 1
    w = torch.full((b, g, cap), 4.0, device="cuda")
    pos = torch.full((b, g, cap), -9, dtype=torch.int32, device="cuda")
    extra = 0 if new is None else 3                        # rows behind the last sequence
    t = sum(counts) + extra
    fused = torch.randn(t, 2 * g + 1, d, generator=_gen(d), device="cuda").to(dt)
    k, v = fused[:, :g], fused[:, g: 2 * g]
    cu = None if new is None else torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    want = [x.clone() for x in (kp, vp, w, pos)]
    at = 0
    for i in range(b):
        for j in range(counts[i]):
            s = past[i] + j
            page = int(table[i, s // size])
            want[0][page, s % size], want[1][page, s % size] = k[at], v[at]
            want[2][i, :, s], want[3][i, :, s] = 0.0, past[i] + 1000 + j
            at += 1
    ops.paged_append(k, v, kp, vp, table, lens, cu_seqlens=cu, seen=seen, weights=w, positions=pos)
    ops.check_status(kp.device)
    for got, ref in zip((kp, vp, w, pos), want):
        assert torch.equal(got, ref)
    assert lens.tolist() == past


@gpu
def test_append_takes_pages_of_any_strides():
    from project_chronos_b200 import ops
    g, d, size = 2, 64, 16
    both = torch.zeros(6, 2, g, size, d, dtype=BF, device="cuda")
    kp, vp = both[:, 0].permute(0, 2, 1, 3), both[:, 1].permute(0, 2, 1, 3)
    table = torch.tensor([[4, 1], [3, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([15, 30], dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, g, d, device="cuda").to(BF), torch.randn(2, g, d, device="cuda").to(BF)
    ops.paged_append(k, v, kp, vp, table, lens)
    assert torch.equal(both[4, 0, :, 15], k[0]) and torch.equal(both[0, 1, :, 14], v[1])
    assert int((both != 0).any(-1).sum()) == 2 * 2 * g


# ---------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------

def _evict_plan(w, pos, n, seen, budget, sinks, recent):
    """src of one (sequence, kv head), by the definition: NaN above every number, ties by the lower slot."""
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)

    def rank(j):
        if pos[j] < sinks or pos[j] >= seen - recent:
            return (0, 0.0, j)
        return (1, 0.0, j) if math.isnan(w[j]) else (2, -w[j], j)

    kept = set(sorted(range(n), key=rank)[:budget])
    movers = iter(sorted(j for j in kept if j >= budget))
    return [j if j in kept else next(movers) for j in range(budget)]


@gpu
@pytest.mark.parametrize("lens, budget, sinks, recent", [
    ([100, 1, 0, 64, 65, 300], 64, 4, 16), ([5, 3, 2], 1, 0, 0), ([5, 3, 2], 1, 1, 0), ([2049, 2050, 1000], 2048, 4, 256),
    ([4000, 3500], 1000, 0, 1000), ([4000, 3500], 1000, 0, 0), ([777], 776, 4, 700), ([1030, 5000], 33, 16, 17)])
@pytest.mark.parametrize("values", ["random", "ties", "special"])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_keeps_the_largest_weights(lens, budget, sinks, recent, values, in_place):
    from project_chronos_b200 import ops
    g, d, size = 2, 16, 16
    kp, vp, table, ln, rows = _make_cache(lens, g, d, size, BF, seed=budget, bad=-1.0)
    b, cap = len(lens), table.shape[1] * size
    gen = _gen(sinks + recent)
    w = torch.exp(3 * torch.randn(b, g, cap, generator=gen, device="cuda"))
    if values == "ties":
        w = torch.randint(0, 3, w.shape, generator=gen, device="cuda").float() - 1.0
        w = torch.where(w == 0, torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.5, -0.0, 0.0), w)
    elif values == "special":
        x = torch.rand(w.shape, generator=gen, device="cuda")
        for lo, val in ((0.0, math.nan), (0.1, math.inf), (0.2, -math.inf), (0.3, 1e-44), (0.4, -1.0), (0.5, 3e38)):
            w = torch.where((x >= lo) & (x < lo + 0.05), torch.full_like(w, val), w)
    # a permutation per head, as earlier evictions leave it, with gaps
    pos = torch.stack([torch.stack([torch.randperm(cap, generator=gen, device="cuda") * 2 for _ in range(g)])
                       for _ in range(b)]).to(torch.int32)
    for i, n in enumerate(lens):   # the positions in use: below seen
        for j in range(g):
            pos[i, j, :n] = (torch.randperm(n, generator=gen, device="cuda") * 3 // 2).to(torch.int32) if n else pos[i, j, :n]
    seen = torch.tensor([max(1, 3 * n // 2) for n in lens], dtype=torch.int32, device="cuda")
    k0, v0, w0, p0 = kp.clone(), vp.clone(), w.clone(), pos.clone()
    wo, po = (None, None) if in_place else (torch.full_like(w, 8.0), torch.full_like(pos, 8))
    r = ops.paged_evict(kp, vp, table, ln, seen, w, pos, budget, sinks=sinks, recent=recent, weights_out=wo, positions_out=po,
                        lens_out=ln if in_place else None)
    ops.check_status(kp.device)
    assert r["lens"].tolist() == [min(n, budget) for n in lens]
    k_want, v_want = k0.clone(), v0.clone()
    for i, n in enumerate(lens):
        t = table[i].long()
        for j in range(g):
            src = _evict_plan(w0[i, j].tolist(), p0[i, j].tolist(), n, int(seen[i]), budget, sinks, recent)
            assert r["src"][i, j].tolist() == src
            m = min(n, budget)
            s = torch.tensor(src[:m], device="cuda", dtype=torch.long)
            to = torch.arange(m, device="cuda")
            assert torch.equal(r["weights"][i, j, :m].view(torch.int32), w0[i, j][s].view(torch.int32))
            assert torch.equal(r["positions"][i, j, :m], p0[i, j][s])
            rest = (w0[i, j, m:], p0[i, j, m:]) if in_place else (torch.full_like(w0[i, j, m:], 8.0), torch.full_like(p0[i, j, m:], 8))
            assert torch.equal(r["weights"][i, j, m:].view(torch.int32), rest[0].view(torch.int32))
            assert torch.equal(r["positions"][i, j, m:], rest[1])
            k_want[t[to // size], to % size, j] = k0[t[s // size], s % size, j]
            v_want[t[to // size], to % size, j] = v0[t[s // size], s % size, j]
    assert torch.equal(kp, k_want) and torch.equal(vp, v_want)
    assert ln.tolist() == ([min(n, budget) for n in lens] if in_place else lens)


@gpu
@pytest.mark.parametrize("dt, d", [(BF, 37), (FP, 5), (FP, 64)])
def test_evict_long_rows_and_any_row_width(dt, d):
    """More slots than shared memory holds keys of; rows copied element by element."""
    from project_chronos_b200 import ops
    n, g, size, budget = 60001, 1, 64, 20000
    width = -(-n // size)
    table = torch.randperm(width, generator=_gen(1), device="cuda").view(1, width).to(torch.int32)
    kp = torch.randn(width, size, g, d, generator=_gen(2), device="cuda").to(dt)
    vp = torch.randn(width, size, g, d, generator=_gen(3), device="cuda").to(dt)
    w = torch.rand(1, g, width * size, generator=_gen(4), device="cuda")
    pos = torch.arange(width * size, dtype=torch.int32, device="cuda").view(1, 1, -1).contiguous()
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    k0, v0 = kp.clone(), vp.clone()
    r = ops.paged_evict(kp, vp, table, ln, ln, w, pos, budget, sinks=3, recent=99, weights_out=torch.empty_like(w),
                        positions_out=torch.empty_like(pos))
    src = _evict_plan(w[0, 0].tolist(), pos[0, 0].tolist(), n, n, budget, 3, 99)
    assert r["src"][0, 0].tolist() == src
    s, to, t = torch.tensor(src, device="cuda"), torch.arange(budget, device="cuda"), table[0].long()
    assert torch.equal(kp[t[to // size], to % size], k0[t[s // size], s % size])
    assert torch.equal(vp[t[to // size], to % size], v0[t[s // size], s % size])


# ---------------------------------------------------------------------------------------
# prompt attention
# ---------------------------------------------------------------------------------------

def _check_prompt(got, lse, q, k, v, lq, lk, cq, ck, window, sinks, dt, rows=None):
    h, d = q.shape[1], q.shape[2]
    for i in (range(lq) if rows is None else rows):
        t = lk - lq + i
        seen = _visible(lk, window, sinks, "cuda", at=t)
        ref, rl, _, a, f = _attend(q[cq + i], k[ck: ck + lk], v[ck: ck + lk], d ** -0.5, seen)
        _check_out(got[cq + i], ref, a, f, lk, dt)
        if lse is not None:
            _check_lse(lse[cq + i], rl, f)


def _some_rows(n):
    return sorted({i for i in (0, 1, 2, n // 3, n // 2, n - 2, n - 1, 31, 32, 63, 64, 127, 128, 129, 255, 256) if 0 <= i < n})


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d", [(8, 2, 128), (4, 4, 64), (6, 2, 80), (5, 1, 128), (16, 1, 96), (2, 1, 256), (3, 1, 37),
                                     (32, 2, 64), (4, 2, 8)])
@pytest.mark.parametrize("lq, past", [([1, 130, 0, 64, 300], [0, 0, 0, 0, 0]), ([3, 129, 40], [500, 1, 127]), ([9, 200], [-4, -150])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 0), (130, 5), (1, 0), (40, 200)])
def test_prompt_attention_matches_its_definition(dt, h, g, d, lq, past, window, sinks):
    from project_chronos_b200 import ops
    lk = [max(0, a + b) for a, b in zip(lq, past)]
    pad = 3
    tq, tk = sum(lq) + pad, sum(lk) + pad
    gen = _gen(h + d)
    q = (2 * torch.randn(tq, h, d, generator=gen, device="cuda")).to(dt)
    k = torch.randn(tk, g, d, generator=gen, device="cuda").to(dt)
    v = torch.randn(tk, g, d, generator=gen, device="cuda").to(dt)
    q[sum(lq):], k[sum(lk):], v[sum(lk):] = math.nan, math.nan, math.inf
    cq = [0] + torch.tensor(lq).cumsum(0).tolist()
    ck = [0] + torch.tensor(lk).cumsum(0).tolist()
    out = torch.full_like(q, 5.0)
    lse = torch.full((tq, h), 5.0, device="cuda")
    ops.window_attention(q, k, v, torch.tensor(cq, dtype=torch.int32, device="cuda"),
                         cu_seqlens_k=torch.tensor(ck, dtype=torch.int32, device="cuda"), window=window, sinks=sinks,
                         out=out, lse=lse)
    ops.check_status(q.device)
    assert bool((out[sum(lq):] == 5.0).all()) and bool((lse[sum(lq):] == 5.0).all())
    for b in range(len(lq)):
        _check_prompt(out, lse, q, k, v, lq[b], lk[b], cq[b], ck[b], window, sinks, dt, _some_rows(lq[b]))


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("window, sinks", [(0, 0), (300, 4), (1000, 130)])
def test_long_prompt_every_tile(dt, window, sinks):
    """Many key tiles per row; every row against the definition, in blocks."""
    from project_chronos_b200 import ops
    n, h, g, d = 2100, 4, 1, 128
    gen = _gen(window)
    qkv = torch.randn(n, h + 2 * g, d, generator=gen, device="cuda")
    qkv[:, :h] *= 3
    qkv = qkv.to(dt)
    q, k, v = qkv[:, :h], qkv[:, h: h + g], qkv[:, h + g:]
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    lse = torch.empty(n, h, device="cuda")
    out = ops.window_attention(q, k, v, cu, window=window, sinks=sinks, lse=lse)
    assert torch.equal(out, ops.window_attention(q, k, v, cu, window=window, sinks=sinks))
    t, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = j <= t
    if window:
        seen = seen & ((j > t - window) | (j < sinks))
    kd, vd = k[:, 0].double(), v[:, 0].double()
    for hh in range(h):
        x = (q[:, hh].double() @ kd.T * d ** -0.5).masked_fill(~seen, -math.inf)
        rl = torch.logsumexp(x, 1)
        p = torch.exp(x - rl[:, None])
        s = (q[:, hh].double().abs() @ kd.abs().T * d ** -0.5).amax(1)
        f = d * 2.0 ** -23 * s + n * 2.0 ** -24 + 2.0 ** -20
        _check_out(out[:, hh], p @ vd, p @ vd.abs(), f, n, dt)
        _check_lse(lse[:, hh], rl, f)


@gpu
@pytest.mark.parametrize("dt, d", [(BF, 128), (HF, 64), (FP, 64)])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_hidden_values_do_not_reach_a_row(dt, d, what):
    """Keys and values that are not finite, at places that some rows see and others do not."""
    from project_chronos_b200 import ops
    n, h, g, window, sinks = 700, 4, 2, 200, 3
    gen = _gen(d)
    q = torch.randn(n, h, d, generator=gen, device="cuda").to(dt)
    k = torch.randn(n, g, d, generator=gen, device="cuda").to(dt)
    v = torch.randn(n, g, d, generator=gen, device="cuda").to(dt)
    at = 300
    v[at, :, 5] = what
    k[at + 1, 0, 7] = math.nan
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = ops.window_attention(q, k, v, cu, window=window, sinks=sinks)
    for i in (0, 100, 250, 298, 299):                     # before: finite and right
        _check_prompt(out, None, q, k, v, n, n, 0, 0, window, sinks, dt, [i])
    for i in (at + window + 1, 600, n - 1):               # behind the window again
        _check_prompt(out, None, q, k, v, n, n, 0, 0, window, sinks, dt, [i])
    for i in (at + 1, at + 60, at + 130, at + window - 1):   # they see it
        group1 = out[i, h // g:]
        assert bool(torch.isnan(out[i, : h // g]).all())
        assert not bool(torch.isfinite(group1[:, 5]).any())
        assert bool(torch.isfinite(group1[:, :5]).all()) and bool(torch.isfinite(group1[:, 6:]).all())


@gpu
def test_prompt_attention_refuses_wrong_tensors():
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    q, k = torch.zeros(9, 4, 64, dtype=BF, device="cuda"), torch.zeros(9, 2, 64, dtype=BF, device="cuda")
    cu = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    ok = dict(q=q, k=k, v=k, cu_seqlens=cu)
    for change in (dict(k=k.half()), dict(v=k[:8]), dict(k=k[:8], v=k[:8]), dict(q=q[..., :32]), dict(cu_seqlens=cu.long()),
                   dict(cu_seqlens_k=cu[:1]), dict(out=q.float()), dict(lse=torch.zeros(9, 3, device="cuda")),
                   dict(v=k.cpu()), dict(cu_seqlens=cu[:0])):
        with pytest.raises((TypeError, ValueError)):
            ops.window_attention(**{**ok, **change})
    with pytest.raises(RuntimeError, match="heads"):
        ops.window_attention(**{**ok, "q": q[:, :3]})
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.window_attention(**{**ok, "k": k.clone().requires_grad_()})
    # offsets that leave the tensors: reported, nothing outside is read or written
    for bad in ([0, 12], [5, 20], [-3, 6]):
        ops.window_attention(q, k, k, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(q.device)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_calls_follow_the_current_stream(dt):
    from project_chronos_b200 import ops
    n, h, g, d = 400, 4, 2, 64
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(20_000_000)
        q = torch.randn(n, h, d, device="cuda").to(dt)
        k, v = torch.randn(n, g, d, device="cuda").to(dt), torch.randn(n, g, d, device="cuda").to(dt)
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        out = ops.window_attention(q, k, v, cu)
        kp, vp = torch.zeros(30, 16, g, d, dtype=dt, device="cuda"), torch.zeros(30, 16, g, d, dtype=dt, device="cuda")
        table = torch.arange(30, dtype=torch.int32, device="cuda").view(1, 30)
        ops.paged_append(k, v, kp, vp, table, torch.zeros(1, dtype=torch.int32, device="cuda"), cu_seqlens=cu)
        one = ops.paged_attn_decode(q[n - 1:], kp, vp, table, torch.full((1,), n, dtype=torch.int32, device="cuda"))
    st.synchronize()
    _check_prompt(out, None, q, k, v, n, n, 0, 0, 0, 0, dt, [0, 200, n - 1])
    ref, _, _, a, f = _attend(q[n - 1], k, v, d ** -0.5, _visible(n, 0, 0, "cuda"))
    _check_out(one[0], ref, a, f, n, dt)


# ---------------------------------------------------------------------------------------
# together: prompt, append, decode steps with running sums, eviction, more steps
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_a_serving_run(dt):
    """A ragged batch is prefilled, decoded, evicted to a budget every few steps; a list
    of the rows that should be there is kept per (sequence, kv head) in 64 bits."""
    from project_chronos_b200 import ops
    h, g, d, size, budget, sinks, recent = 8, 2, 64, 16, 48, 2, 16
    prompts, steps = [70, 5, 33], 24
    b = len(prompts)
    gen = _gen(77)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    width = 8
    kp, vp = (torch.full((b * width, size, g, d), math.nan, dtype=dt, device="cuda") for _ in range(2))
    table = torch.randperm(b * width, generator=gen, device="cuda").view(b, width).to(torch.int32)
    w = torch.full((b, g, width * size), math.nan, device="cuda")
    pos = torch.full((b, g, width * size), -1, dtype=torch.int32, device="cuda")
    lens, seen = (torch.zeros(b, dtype=torch.int32, device="cuda") for _ in range(2))
    t = sum(prompts)
    cu = torch.tensor([0] + torch.tensor(prompts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    q, k, v = rnd(t, h, d), rnd(t, g, d), rnd(t, g, d)
    out = ops.window_attention(q, k, v, cu)
    for i, n in enumerate(prompts):
        _check_prompt(out, None, q, k, v, n, n, int(cu[i]), int(cu[i]), 0, 0, dt, _some_rows(n))
    ops.paged_append(k, v, kp, vp, table, lens, cu_seqlens=cu, seen=seen, weights=w, positions=pos)
    lens += cu.diff()
    seen += cu.diff()
    book = [[[[k[int(cu[i]) + j, x], v[int(cu[i]) + j, x], 0.0, j] for j in range(prompts[i])] for x in range(g)]
            for i in range(b)]
    for step in range(steps):
        q, k, v = rnd(b, h, d), rnd(b, g, d), rnd(b, g, d)
        ops.paged_append(k, v, kp, vp, table, lens, seen=seen, weights=w, positions=pos)
        lens += 1
        seen += 1
        out = ops.paged_attn_decode(q, kp, vp, table, lens, weights=w)
        for i in range(b):
            for x in range(g):
                rows = book[i][x]
                rows.append([k[i, x], v[i, x], 0.0, int(seen[i]) - 1])
                ks, vs = torch.stack([r[0] for r in rows])[:, None], torch.stack([r[1] for r in rows])[:, None]
                part = slice(x * h // g, (x + 1) * h // g)
                ref, _, p, a, f = _attend(q[i, part], ks, vs, d ** -0.5, _visible(len(rows), 0, 0, "cuda"))
                _check_out(out[i, part], ref, a, f, len(rows), dt)
                for r, y in zip(rows, p.sum(0).tolist()):
                    r[2] += y
        if step % 5 == 4:
            # the kernel's own sums decide (they differ from the 64-bit ones by rounding); they are checked first
            for i in range(b):
                for x in range(g):
                    mine = torch.tensor([r[2] for r in book[i][x]], device="cuda", dtype=torch.float64)
                    got = w[i, x, : len(mine)].double()
                    assert bool(((got - mine).abs() <= 1e-3 * mine).all())   # up to 24 steps of f <= D 2^-23 S each
            plans = [[_evict_plan(w[i, x].tolist(), pos[i, x].tolist(), int(lens[i]), int(seen[i]), budget, sinks, recent)
                      for x in range(g)] for i in range(b)]
            r = ops.paged_evict(kp, vp, table, lens, seen, w, pos, budget, sinks=sinks, recent=recent, lens_out=lens)
            for i in range(b):
                for x in range(g):
                    assert r["src"][i, x].tolist() == plans[i][x]
                    book[i][x] = [book[i][x][j] for j in plans[i][x] if j >= 0]
                    assert [y[3] for y in book[i][x]] == pos[i, x, : len(book[i][x])].tolist()
    ops.check_status(kp.device)


@gpu
def test_paged_cache_rows_come_and_go():
    """The cache object: a row ends, its pages serve another one; a row without pages is
    refused on the device; a captured step replays while the rows grow."""
    from project_chronos_b200 import PagedCache, ops
    from project_chronos_b200 import _native as N
    h, g, d, dt = 8, 2, 64, BF
    gen = _gen(5)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    c = PagedCache(2, 12, g, d, 8, "cuda", dt, page_size=16, track_weights=True)
    book = [[], []]

    def step(one):
        k, v, q = rnd(2, g, d), rnd(2, g, d), rnd(2, h, d)
        c.append(k, v)
        out = one(q)
        for b in range(2):
            book[b].append((k[b], v[b]))
            ks, vs = (torch.stack([r[i] for r in book[b]]) for i in (0, 1))
            ref, _, _, a, f = _attend(q[b], ks, vs, d ** -0.5, _visible(len(ks), 0, 0, "cuda"))
            _check_out(out[b], ref, a, f, len(ks), dt)

    for b, n in enumerate((40, 7)):
        c.reserve(b, n + 40)
    k, v = rnd(47, g, d), rnd(47, g, d)
    c.append(k, v, torch.tensor([0, 40, 47], dtype=torch.int32, device="cuda"))
    book[0] = [(k[i], v[i]) for i in range(40)]
    book[1] = [(k[i], v[i]) for i in range(40, 47)]
    step(c.attend)
    static_q, static_out = rnd(2, h, d), torch.empty(2, h, d, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(static_q, out=static_out)

    def replay(q):
        static_q.copy_(q)
        graph.replay()
        return static_out

    for _ in range(20):
        step(replay)
    # row 0 ends; its pages go to row 1, which goes on, and a new row 0 starts
    c.release(0)
    book[0] = []
    c.reserve(1, 100)
    c.reserve(0, 60)
    for _ in range(25):
        step(replay)
    ops.check_status(c.lens.device)
    assert c.positions[0, 0, :25].tolist() == list(range(25))
    q = rnd(2, h, d)
    assert bool(torch.isfinite(c.attend(q, window=20, sinks=2)).all())
    src = c.evict(20, sinks=2, recent=8)
    assert c.lens.tolist() == [20, 20] and sorted(src[0, 0].tolist())[:2] == [0, 1]
    with pytest.raises(RuntimeError, match="window"):
        c.attend(q, window=20)
    c.release(0)
    with pytest.raises(RuntimeError, match="at most 8"):
        c.reserve(1, 128 * 2)
    c.append(rnd(2, g, d), rnd(2, g, d))                 # row 0 has no pages
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(c.lens.device)


# ---------------------------------------------------------------------------------------
# many rows, other strides, captured evictions
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt, d", [(BF, 128), (BF, 64), (FP, 128), (HF, 256)])
@pytest.mark.parametrize("b, most", [(400, 60), (400, 200), (150, 500), (70, 1500)])
def test_decode_of_many_rows(dt, d, b, most):
    """Around the choice between clusters and the work list: more rows than blocks, rows of
    one to many blocks, none at all."""
    from project_chronos_b200 import ops
    gen = torch.Generator().manual_seed(b + most)
    lens = torch.randint(0, most + 1, (b,), generator=gen).tolist()
    lens[:3] = [0, most, 1]
    h, g = 6, 2
    kp, vp, table, ln, rows = _make_cache(lens, g, d, 16, dt, seed=d)
    q = (2 * torch.randn(b, h, d, generator=_gen(1), device="cuda")).to(dt)
    lse = torch.empty(b, h, device="cuda")
    out = ops.paged_attn_decode(q, kp, vp, table, ln, scale=0.11, lse=lse)
    for i in list(range(0, b, 17)) + [1, 2, b - 1]:
        k, v = rows[i]
        ref, rl, _, a, f = _attend(q[i], k, v, 0.11, _visible(lens[i], 0, 0, "cuda"))
        _check_out(out[i], ref, a, f, lens[i], dt)
        _check_lse(lse[i], rl, f)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_many_short_sequences(dt):
    from project_chronos_b200 import ops
    b, h, g, d, size = 1100, 4, 2, 64, 16
    gen = torch.Generator().manual_seed(3)
    new = torch.randint(0, 9, (b,), generator=gen).tolist()
    t = sum(new)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    q = torch.randn(t, h, d, generator=_gen(1), device="cuda").to(dt)
    k, v = (torch.randn(t, g, d, generator=_gen(2 + i), device="cuda").to(dt) for i in range(2))
    out = ops.window_attention(q, k, v, cu, window=3, sinks=1)
    kp, vp = (torch.zeros(b, size, g, d, dtype=dt, device="cuda") for _ in range(2))
    table = torch.randperm(b, generator=_gen(9), device="cuda").to(torch.int32).view(b, 1)
    ops.paged_append(k, v, kp, vp, table, torch.zeros(b, dtype=torch.int32, device="cuda"), cu_seqlens=cu)
    last = torch.tensor([max(0, int(cu[i + 1]) - 1) for i in range(b)], device="cuda")
    one = ops.paged_attn_decode(q[last].contiguous(), kp, vp, table, cu.diff().contiguous(), window=3, sinks=1)
    ops.check_status(q.device)
    for i in range(0, b, 29):
        n, c0 = new[i], int(cu[i])
        _check_prompt(out, None, q, k, v, n, n, c0, c0, 3, 1, dt)
        if n:
            assert torch.equal(kp[int(table[i, 0]), :n], k[c0: c0 + n])
            ref, _, _, a, f = _attend(q[c0 + n - 1], k[c0: c0 + n], v[c0: c0 + n], d ** -0.5, _visible(n, 3, 1, "cuda"))
            _check_out(one[i], ref, a, f, n, dt)
        else:
            assert bool((one[i] == 0).all())


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("layout", ["fused", "heads first", "odd strides"])
def test_prompt_attention_takes_strides(dt, layout):
    from project_chronos_b200 import ops
    n, h, g, d = 300, 6, 2, 64
    x = torch.randn(n, h + 2 * g, d, generator=_gen(4), device="cuda").to(dt)
    if layout == "heads first":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "odd strides":
        x = torch.cat([x, x[..., :1]], dim=-1)[..., :d]
    q, k, v = x[:, :h], x[:, h: h + g], x[:, h + g:]
    wide = torch.full((n, h + 1, d + (1 if layout == "odd strides" else 8)), 3.0, dtype=dt, device="cuda")
    cu = torch.tensor([0, 100, n], dtype=torch.int32, device="cuda")
    ops.window_attention(q, k, v, cu, out=wide[:, :h, :d], window=90, sinks=2)
    for c0, m in ((0, 100), (100, 200)):
        _check_prompt(wide[:, :h, :d], None, q, k, v, m, m, c0, c0, 90, 2, dt, _some_rows(m))
    assert bool((wide[:, h:] == 3.0).all()) and bool((wide[..., d:] == 3.0).all())


@gpu
@pytest.mark.parametrize("n, budget", [(900, 820), (900, 300)])
def test_captured_evictions(n, budget):
    """One kernel (few slots) and two, replayed on new contents; a row shorter than the budget."""
    from project_chronos_b200 import ops
    g, d, size = 2, 32, 16
    kp, vp, table, ln, _ = _make_cache([n, 20], g, d, size, BF, seed=1, width=-(-n // size), bad=0.0)
    cap = table.shape[1] * size
    w = torch.zeros(2, g, cap, device="cuda")
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(2, g, cap).contiguous()
    wo, po = torch.zeros_like(w), torch.zeros_like(pos)
    call = lambda: ops.paged_evict(kp, vp, table, ln, ln, w, pos, budget, sinks=2, recent=9, weights_out=wo, positions_out=po)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = call()
    for seed in range(3):
        kp.copy_(torch.randn(kp.shape, generator=_gen(seed), device="cuda"))
        vp.copy_(torch.randn(vp.shape, generator=_gen(seed + 9), device="cuda"))
        w.copy_(torch.rand(w.shape, generator=_gen(seed + 20), device="cuda"))
        k0, v0 = kp.clone(), vp.clone()
        graph.replay()
        assert r["lens"].tolist() == [budget, 20]
        t = table[0].long()
        for j in range(g):
            src = _evict_plan(w[0, j].tolist(), pos[0, j].tolist(), n, n, budget, 2, 9)
            assert r["src"][0, j].tolist() == src
            s, to = torch.tensor(src, device="cuda"), torch.arange(budget, device="cuda")
            assert torch.equal(kp[t[to // size], to % size, j], k0[t[s // size], s % size, j])
            assert torch.equal(vp[t[to // size], to % size, j], v0[t[s // size], s % size, j])
        assert torch.equal(kp[table[1].long()], k0[table[1].long()])


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_the_longest_windows(dt):
    """A window of 2^31 - 1 hides nothing, whatever the position; more is refused."""
    from project_chronos_b200 import ops
    big = 2 ** 31 - 1
    h, g, d = 4, 2, 64
    gen = _gen(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    q, k, v = rnd(370, h, d), rnd(270, g, d), rnd(270, g, d)   # the first 100 rows see nothing
    cq, ck = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 300, 370], [0, 200, 270]))
    for window, sinks in ((big, 0), (big, big), (3, big)):
        out = ops.window_attention(q, k, v, cq, cu_seqlens_k=ck, window=window, sinks=sinks)
        _check_prompt(out, None, q, k, v, 300, 200, 0, 0, 0, 0, dt, [0, 99, 100, 101, 299])
        _check_prompt(out, None, q, k, v, 70, 70, 300, 200, 0, 0, dt, [0, 69])
    kp, vp, table, ln, rows = _make_cache([90, 1], g, d, 16, dt, seed=3)
    q1 = rnd(2, h, d)
    for window, sinks in ((big, 0), (big, big), (3, big)):
        out = ops.paged_attn_decode(q1, kp, vp, table, ln, window=window, sinks=sinks)
        for b, (kk, vv) in enumerate(rows):
            ref, _, _, a, f = _attend(q1[b], kk, vv, d ** -0.5, _visible(len(kk), 0, 0, "cuda"))
            _check_out(out[b], ref, a, f, len(kk), dt)
    for bad in (dict(window=2 ** 31), dict(window=2 ** 32 + 3), dict(sinks=2 ** 40), dict(window=-2 ** 31 - 1)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.paged_attn_decode(q1, kp, vp, table, ln, **bad)
        with pytest.raises(ValueError, match="32 bits"):
            ops.window_attention(q, k, v, cq, cu_seqlens_k=ck, **bad)
    with pytest.raises(RuntimeError, match="negative"):
        ops.paged_attn_decode(q1, kp, vp, table, ln, window=-5)


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("d", [64, 36])
def test_decode_passes_on_what_is_not_finite(dt, d):
    """A visible NaN or infinity reaches the heads (columns) that read it, a hidden one none."""
    from project_chronos_b200 import ops
    h, g = 4, 2
    kp, vp, table, ln, rows = _make_cache([200, 200, 200], g, d, 16, dt, seed=3)
    q = torch.randn(3, h, d, generator=_gen(1), device="cuda").to(dt)
    at = lambda b, s: (int(table[b, s // 16]), s % 16)  # noqa: E731
    kp[at(0, 77)][0, 3] = math.nan
    vp[at(1, 77)][1, 5] = math.inf
    vp[at(2, 10)][:, :] = math.nan                    # hidden by the window
    kp[at(2, 11)][:, :] = math.inf
    out = ops.paged_attn_decode(q, kp, vp, table, ln, window=150, sinks=4)
    assert bool(torch.isnan(out[0, :2]).all()) and bool(torch.isfinite(out[0, 2:]).all())
    assert bool((out[1, 2:, 5] == math.inf).all())
    assert bool(torch.isfinite(out[1, :2]).all()) and bool(torch.isfinite(out[1, 2:, :5]).all())
    k, v = rows[2]
    ref, _, _, a, f = _attend(q[2], k, v, d ** -0.5, _visible(200, 150, 4, "cuda"))
    _check_out(out[2], ref, a, f, 200, dt)


@gpu
def test_empty_calls_on_the_device():
    from project_chronos_b200 import ops
    z = dict(dtype=BF, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    kp = torch.zeros(3, 16, 2, 64, **z)
    none = ops.paged_attn_decode(torch.zeros(0, 4, 64, **z), kp, kp, torch.zeros(0, 2, **i32), torch.zeros(0, **i32))
    assert none.shape == (0, 4, 64)
    # no pages at all: every row is empty
    no = torch.zeros(0, 16, 2, 64, **z)
    out = ops.paged_attn_decode(torch.ones(2, 4, 64, **z), no, no, torch.zeros(2, 0, **i32), torch.zeros(2, **i32))
    assert bool((out == 0).all())
    assert ops.window_attention(torch.zeros(0, 4, 64, **z), torch.zeros(5, 2, 64, **z), torch.zeros(5, 2, 64, **z),
                                torch.zeros(2, **i32), cu_seqlens_k=torch.zeros(2, **i32)).shape == (0, 4, 64)
    # queries without keys see nothing
    lse = torch.zeros(3, 4, device="cuda")
    out = ops.window_attention(torch.ones(3, 4, 64, **z), torch.zeros(0, 2, 64, **z), torch.zeros(0, 2, 64, **z),
                               torch.tensor([0, 3], **i32), cu_seqlens_k=torch.zeros(2, **i32), lse=lse)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    ops.paged_append(torch.zeros(0, 2, 64, **z), torch.zeros(0, 2, 64, **z), kp, kp.clone(), torch.zeros(1, 1, **i32),
                     torch.zeros(1, **i32), cu_seqlens=torch.zeros(2, **i32))
    w = torch.zeros(1, 2, 16, device="cuda")
    r = ops.paged_evict(kp, kp.clone(), torch.zeros(1, 1, **i32), torch.zeros(1, **i32), torch.zeros(1, **i32), w,
                        torch.zeros(1, 2, 16, **i32), 40)
    assert r["lens"].tolist() == [0] and bool((r["src"] == -1).all())
    ops.check_status(kp.device)


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("h, g, d", [(8, 2, 128), (4, 4, 64), (6, 1, 80)])
@pytest.mark.parametrize("lq, past", [([1], [3000]), ([64], [5000]), ([130], [2500]), ([3, 3], [9000, 2]), ([5, 0, 200], [1700, 4000, 1500])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1900, 150), (60, 3)])
def test_few_queries_on_many_keys(dt, h, g, d, lq, past, window, sinks):
    """Row tiles whose keys a cluster shares; blocks of it without keys."""
    from project_chronos_b200 import ops
    lk = [a + b for a, b in zip(lq, past)]
    gen = _gen(h + lq[0])
    q = (2 * torch.randn(sum(lq) + 2, h, d, generator=gen, device="cuda")).to(dt)
    k = torch.randn(sum(lk), g, d, generator=gen, device="cuda").to(dt)
    v = torch.randn(sum(lk), g, d, generator=gen, device="cuda").to(dt)
    cq, ck = ([0] + torch.tensor(x).cumsum(0).tolist() for x in (lq, lk))
    out = torch.full_like(q, 5.0)
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    call = lambda o, e: ops.window_attention(  # noqa: E731
        q, k, v, torch.tensor(cq, dtype=torch.int32, device="cuda"), cu_seqlens_k=torch.tensor(ck, dtype=torch.int32, device="cuda"),
        window=window, sinks=sinks, out=o, lse=e)
    call(out, lse)
    again = torch.full_like(q, 5.0)
    call(again, None)
    ops.check_status(q.device)
    assert torch.equal(out, again)
    assert bool((out[sum(lq):] == 5.0).all()) and bool((lse[sum(lq):] == 5.0).all())
    for b in range(len(lq)):
        _check_prompt(out, lse, q, k, v, lq[b], lk[b], cq[b], ck[b], window, sinks, dt, _some_rows(lq[b]))


@gpu
def test_hidden_values_do_not_reach_a_split_row():
    from project_chronos_b200 import ops
    n, past, h, g, d, window = 90, 4000, 8, 2, 128, 3000
    gen = _gen(2)
    q, k, v = (torch.randn(r, x, d, generator=gen, device="cuda").to(BF) for r, x in ((n, h), (n + past, g), (n + past, g)))
    first = past - window + 40                        # seen by the rows up to 39 - 1 only
    v[first, 1, 7] = math.nan
    v[past + 50, :, 3] = math.inf                     # seen from row 50 on
    cq, ck = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (n, n + past))
    out = ops.window_attention(q, k, v, cq, cu_seqlens_k=ck, window=window)
    clean = v.clone()
    clean[first], clean[past + 50] = 0.0, 0.0
    for i in (39, 40, 45, 49):                        # row i sees keys past + i - window + 1 .. past + i
        sees_first = past + i - window < first
        assert sees_first == (i < 40)
        if not sees_first:
            _check_prompt(out, None, q, k, clean, n, n + past, 0, 0, window, 0, BF, [i])
    assert bool(torch.isnan(out[20, 4:, 7]).all()) and bool(torch.isfinite(out[20, :4]).all())
    assert bool((out[60, :, 3] == math.inf).all()) and bool(torch.isfinite(out[60, :, 4:]).all())


# ---------------------------------------------------------------------------------------
# lengths that the append counts
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("track", [True, False])
def test_dropped_tokens_are_not_counted(track):
    """A row without pages, or with too few, keeps the length of what it stored: what comes
    after it gets pages again lands right behind, and nothing stale is attended to."""
    from project_chronos_b200 import PagedCache, ops
    from project_chronos_b200 import _native as N
    h, g, d, dt = 8, 2, 64, BF
    gen = _gen(15)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    c = PagedCache(2, 12, g, d, 8, "cuda", dt, page_size=16, track_weights=track)
    dev = c.lens.device
    book = [[], []]

    def put(counts, stored):
        t = sum(counts)
        k, v = rnd(t, g, d), rnd(t, g, d)
        cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        c.append(k, v, None if counts == [1, 1] else cu)
        at = 0
        for b, n in enumerate(counts):
            book[b] += [(k[at + i], v[at + i]) for i in range(stored[b])]
            at += n
        if list(counts) != list(stored):
            with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
                ops.check_status(dev)
        look()

    def look():
        assert c.lens.tolist() == [len(x) for x in book] and c.seen.tolist() == c.lens.tolist()
        q = rnd(2, h, d)
        out = c.attend(q)
        ops.check_status(dev)
        for b in range(2):
            if track:
                assert c.positions[b, 0, : len(book[b])].tolist() == list(range(len(book[b])))
            if not book[b]:
                assert bool((out[b] == 0).all())
                continue
            ks, vs = (torch.stack([r[i] for r in book[b]]) for i in (0, 1))
            ref, _, _, a, f = _attend(q[b], ks, vs, d ** -0.5, _visible(len(ks), 0, 0, "cuda"))
            _check_out(out[b], ref, a, f, len(ks), dt)

    c.reserve(0, 40)
    c.reserve(1, 60)
    put([40, 20], [40, 20])
    c.release(0)
    book[0] = []
    for _ in range(5):
        put([1, 1], [0, 1])                           # row 0 is idle
    c.reserve(0, 33)                                  # 48 slots, pages used before
    put([33, 0], [33, 0])
    for i in range(18):                               # row 0 is full after 15
        put([1, 1], [int(i < 15), 1])
    c.reserve(0, 64)
    put([1, 1], [1, 1])
    put([40, 2], [15, 2])                             # the first 15 of a packed row fit
    c.reserve(0, 70)
    put([3, 0], [3, 0])


@gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dt, d", [(BF, 64), (FP, 5)])
def test_append_counts_what_it_stored(dt, d, in_place):
    """Lengths and tokens seen after packed and one-token calls: rows that are full, have a hole in
    their table, none of it, a bad length, no tokens."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    g, size, width = 2, 4, 70
    b = 45
    gen = torch.Generator().manual_seed(d)
    have = torch.randint(0, width + 1, (b,), generator=gen)     # pages of each row
    have[:4] = torch.tensor([width, width, 0, 40])
    past = (torch.rand(b, generator=gen) * (have * size + 1)).long().clamp(max=width * size)
    new = torch.randint(0, 60, (b,), generator=gen)
    new[:6] = torch.tensor([width * size, 0, 5, 200, 0, 1])
    past[0], past[3] = 0, 9
    table = torch.full((b, width), -1, dtype=torch.int32)
    pages = int(have.sum())
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    at = 0
    for i in range(b):
        table[i, : have[i]] = order[at: at + int(have[i])]
        at += int(have[i])
    table[3, 35] = pages                                        # a page that is none, its neighbours are
    past[7] = -1
    room = have * size
    room[3], room[7] = 35 * size, -1
    to = dict(dtype=torch.int32, device="cuda")
    for counts in (new, torch.ones(b, dtype=torch.long)):
        kp, vp = (torch.zeros(pages, size, g, d, dtype=dt, device="cuda") for _ in range(2))
        lens, seen = past.to(**to), (past + 1000).to(**to)
        t = int(counts.sum())
        k, v = (torch.randn(t, g, d, generator=_gen(i), device="cuda").to(dt) for i in (1, 2))
        cu = None if counts is not new else torch.tensor([0] + counts.cumsum(0).tolist(), **to)
        lo, so = (lens, seen) if in_place else (torch.full_like(lens, 77), torch.full_like(seen, 77))
        ops.paged_append(k, v, kp, vp, table.cuda(), lens, cu_seqlens=cu, seen=seen, lens_out=lo, seen_out=so)
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(kp.device)
        stored = torch.minimum(counts, (room - past).clamp(min=0))
        stored[7] = 0
        assert lo.tolist() == (past + stored).tolist() and so.tolist() == (past + 1000 + stored).tolist()
        if not in_place:
            assert lens.tolist() == past.tolist()
        first = 0
        for i in range(b):
            for j in range(int(stored[i])):
                s = int(past[i]) + j
                assert torch.equal(kp[int(table[i, s // size]), s % size], k[first + j])
            first += int(counts[i])
    # offsets beyond the rows count what is there; without rows the lengths are copied
    ops.paged_append(k[:3], v[:3], kp, vp, table[:2].cuda(), torch.zeros(2, **to), cu_seqlens=torch.tensor([0, 2, 9], **to),
                     lens_out=lo[:2])
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(kp.device)
    assert lo[:2].tolist() == [2, 1]
    ops.paged_append(k[:0], v[:0], kp, vp, table[:2].cuda(), torch.tensor([5, 6], **to), cu_seqlens=torch.zeros(3, **to),
                     lens_out=lo[:2])
    assert lo[:2].tolist() == [5, 6]
    ops.check_status(kp.device)


def test_append_refuses_lengths_that_overlap(lib):
    from project_chronos_b200 import _native as N
    for f, text in ((dict(seen_out=4096), b"seen_out needs seen"), (dict(lens_out=1028), b"overlap"),
                    (dict(seen=2048, seen_out=2052), b"overlap"), (dict(seen=2048, lens_out=2048), b"overlap"),
                    (dict(seen=2048, seen_out=1024), b"overlap"), (dict(seen=2048, seen_out=4096, lens_out=4100), b"overlap"),
                    (dict(seen=2048, seen_out=2048, lens_out=1024), b"required")):
        a = N.ChronosPagedAppendArgs(cache=_native_cache(N, lens=1024), num_tokens=2, **f)
        assert lib.chronos_paged_append(ctypes.byref(a), None) == N.CHRONOS_ERR_INVALID_ARG
        assert text in lib.chronos_moe_last_error()


# ---------------------------------------------------------------------------------------
# fp16 weights far below the largest
# ---------------------------------------------------------------------------------------

def _fp16_terms(n, v):
    """What rounding to fp16 adds where weights are taken against a maximum 2^7 below: the result's
    last place below the normal range, and the weights' (2^-25 of 2^7, relative to a sum of at least 1)."""
    return 2.0 ** -25 + n * 2.0 ** -32 * float(v.abs().max())


def _check_tight(got, ref, a, f, n, v):
    u = _unit(HF)
    tol = u * ref.abs() + (u + f[:, None] + n * 2.0 ** -23) * a + _fp16_terms(n, v)
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the tolerance"


def _some_heavy(n, g, d, gap, at):
    """Keys and values of which the slots `at` outweigh each other one by 2^gap, for a query whose first
    16 elements sum to `gap`; their values are zero, so the result is what the light ones leave."""
    k = torch.zeros(n, g, d, dtype=HF, device="cuda")
    k[at, :, :16] = math.log(2.0)
    v = (64.0 + 64.0 * torch.rand(n, g, d, generator=_gen(gap), device="cuda")).to(HF)
    v[at] = 0.0
    return k, v


@gpu
@pytest.mark.parametrize("gap", [20, 25, 26, 29])
@pytest.mark.parametrize("b, n, h, g, d", [(1, 131072, 8, 2, 128), (300, 4001, 16, 2, 64), (140, 500, 20, 2, 256), (140, 500, 4, 2, 128),
                                           (2, 9000, 6, 2, 36)])
def test_fp16_light_slots_count_next_to_heavy_ones(b, n, h, g, d, gap):
    """One heavy slot for each of a block's warps; fewer and more rows than blocks."""
    from project_chronos_b200 import ops
    size = 16
    k, v = _some_heavy(n, g, d, gap, [5, 21, 37, 53])
    width = -(-n // size)
    table = torch.arange(width, dtype=torch.int32, device="cuda").expand(b, width).contiguous()
    kp, vp = (torch.zeros(width * size, g, d, dtype=HF, device="cuda") for _ in range(2))
    kp[:n], vp[:n] = k, v
    kp, vp = kp.view(width, size, g, d), vp.view(width, size, g, d)
    q = torch.zeros(b, h, d, dtype=HF, device="cuda")
    q[..., :16] = gap / 16
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    w = torch.zeros(b, g, width * size, device="cuda")
    lse, lse2 = torch.empty(b, h, device="cuda"), torch.empty(b, h, device="cuda")
    out = ops.paged_attn_decode(q, kp, vp, table, lens, scale=1.0, lse=lse)
    out2 = ops.paged_attn_decode(q, kp, vp, table, lens, scale=1.0, lse=lse2, weights=w)
    ref, rl, p, a, f = _attend(q[0], k, v, 1.0, _visible(n, 0, 0, "cuda"))
    want = p.view(g, h // g, n).sum(1)
    for i in (0, b // 2, b - 1):
        for o, e in ((out, lse), (out2, lse2)):
            _check_tight(o[i], ref, a, f, n, v)
            _check_lse(e[i], rl, f)
        assert bool(((w[i, :, :n].double() - want).abs() <= (f.max() + (h + 1) * 2.0 ** -24) * want).all())


@gpu
@pytest.mark.parametrize("gap", [20, 25, 26, 29])
@pytest.mark.parametrize("h, g, d, lq, lk", [(8, 2, 128, 40, 9000), (4, 4, 64, 600, 4000), (4, 1, 128, 1, 20000), (4, 2, 80, 4000, 4000)])
def test_fp16_light_keys_count_next_to_a_heavy_one(h, g, d, lq, lk, gap):
    from project_chronos_b200 import ops
    k, v = _some_heavy(lk, g, d, gap, [5])
    q = torch.zeros(lq, h, d, dtype=HF, device="cuda")
    q[..., :16] = gap / 16
    cq, ck = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (lq, lk))
    lse = torch.empty(lq, h, device="cuda")
    out = ops.window_attention(q, k, v, cq, cu_seqlens_k=ck, scale=1.0, lse=lse)
    for i in _some_rows(lq):
        if lk - lq + i < 6:
            continue
        ref, rl, _, a, f = _attend(q[i], k, v, 1.0, _visible(lk, 0, 0, "cuda", at=lk - lq + i))
        _check_tight(out[i], ref, a, f, lk, v)
        _check_lse(lse[i], rl, f)


@gpu
@pytest.mark.parametrize("step", [7.9, 8.0, 8.1, 15.0])
def test_fp16_scores_that_climb(step):
    """Maxima that lag behind by up to 2^8 in weight, every 128 keys a step higher."""
    from project_chronos_b200 import ops
    n, h, g, d, size = 1000, 8, 2, 64, 16
    k = torch.zeros(n, g, d, dtype=HF, device="cuda")
    k[:, :, 0] = (torch.arange(n, device="cuda") // 128).to(HF)[:, None]
    v = torch.randn(n, g, d, generator=_gen(1), device="cuda").to(HF)
    q = torch.zeros(n, h, d, dtype=HF, device="cuda")
    q[..., 0] = step
    scale = math.log(2.0)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    lse = torch.empty(n, h, device="cuda")
    out = ops.window_attention(q, k, v, cu, scale=scale, lse=lse)
    kp, vp = (torch.zeros(63 * size, g, d, dtype=HF, device="cuda") for _ in range(2))
    kp[:n], vp[:n] = k, v
    table = torch.arange(63, dtype=torch.int32, device="cuda").view(1, 63)
    one = ops.paged_attn_decode(q[n - 1:], kp.view(63, size, g, d), vp.view(63, size, g, d), table, cu[1:], scale=scale)
    for i in _some_rows(n) + [400, 700]:
        ref, rl, _, a, f = _attend(q[i], k, v, scale, _visible(n, 0, 0, "cuda", at=i))
        _check_tight(out[i], ref, a, f, n, v)
        _check_lse(lse[i], rl, f)
        if i == n - 1:
            _check_tight(one[0], ref, a, f, n, v)


# ---------------------------------------------------------------------------------------
# running sums under a table far wider than the rows
# ---------------------------------------------------------------------------------------

def test_score_workspace_is_bounded(lib):
    """Running sums keep scores of a bounded number of sequences at a time, however wide the table is."""
    from project_chronos_b200 import _native as N
    for batch, width in ((64, 2048), (4096, 512), (256, 1 << 14)):
        c = N.ChronosPagedCache(batch=batch, kv_heads=8, head_dim=128, dtype=N.DTYPE_BF16, num_pages=99, page_size=64,
                                table_width=width)
        a = N.ChronosPagedDecodeArgs(cache=c, heads=32, scale=1.0, weights=256, weights_out=256, slot_cap=64 * width)
        n = lib.chronos_paged_decode_workspace(ctypes.byref(a))
        one = 32 * 64 * width * 4                     # a sequence's
        assert 0 < n <= max(1 << 28, one) + (1 << 24)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_summed_weights_under_a_wide_table(dt):
    """Rows far shorter than their table: the call runs over groups of sequences."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    b, h, g, d, size, width = 150, 16, 2, 64, 16, 2048
    gen = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 400, (b,), generator=gen).tolist()
    kp, vp, _, ln, rows = _make_cache(lens, g, d, size, dt, seed=11)
    narrow = _make_cache(lens, g, d, size, dt, seed=11)[2]
    table = torch.full((b, 2 * width), -1, dtype=torch.int32, device="cuda")[:, :width]
    table[:, : narrow.shape[1]] = narrow
    q = (2 * torch.randn(b, h + 1, d, generator=_gen(9), device="cuda")).to(dt)[:, :h]
    w0 = torch.rand(b, g, width * size, generator=_gen(10), device="cuda")
    for window, sinks in ((0, 0), (90, 3)):
        w = w0.clone()
        lse = torch.empty(b, h, device="cuda")
        wide = torch.full((b, h + 1, d), 9.0, dtype=dt, device="cuda")
        ops.paged_attn_decode(q, kp, vp, table, ln, window=window, sinks=sinks, weights=w, lse=lse, out=wide[:, :h])
        ops.check_status(kp.device)
        assert bool((wide[:, h] == 9.0).all())
        again = w0.clone()
        assert torch.equal(wide[:, :h], ops.paged_attn_decode(q, kp, vp, table, ln, window=window, sinks=sinks, weights=again))
        assert torch.equal(w, again)
        for i in range(b):
            k, v = rows[i]
            n = lens[i]
            ref, rl, p, a, f = _attend(q[i], k, v, d ** -0.5, _visible(n, window, sinks, "cuda"))
            _check_out(wide[i, :h], ref, a, f, n, dt)
            _check_lse(lse[i], rl, f)
            add = p.view(g, h // g, n).sum(1)
            want = w0[i, :, :n].double() + add
            tol = f.view(g, h // g).amax(1)[:, None] * add + (h // g + 1) * 2.0 ** -24 * want
            assert bool(((w[i, :, :n].double() - want).abs() <= tol).all())
            assert torch.equal(w[i, :, n:], w0[i, :, n:])
    ln[b - 1] = width * size + 5
    ops.paged_attn_decode(q, kp, vp, table, ln, weights=w0)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(kp.device)


# ---------------------------------------------------------------------------------------
# windows and evictions
# ---------------------------------------------------------------------------------------

def test_a_refused_eviction_leaves_the_window():
    from project_chronos_b200 import PagedCache
    c = PagedCache(1, 4, 1, 8, 4, "cpu", torch.float32, page_size=4, track_weights=True)
    c.reserve(0, 9)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.evict(4)
    with pytest.raises(RuntimeError, match="CUDA"):   # not "a window counts slots"
        c.attend(torch.zeros(1, 1, 8), window=3)


@gpu
def test_windows_come_back_after_evictions():
    """A window is refused while a row that an eviction cut lives, and only then."""
    from project_chronos_b200 import PagedCache, ops
    h, g, d, dt, window, sinks = 8, 2, 64, BF, 20, 2
    gen = _gen(6)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dt)  # noqa: E731
    c = PagedCache(2, 20, g, d, 8, "cuda", dt, page_size=16, track_weights=True)
    lens = [50, 9]

    def fill():
        k, v = rnd(sum(lens), g, d), rnd(sum(lens), g, d)
        c.append(k, v, torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda"))
        return [(k[: lens[0]], v[: lens[0]]), (k[lens[0]:], v[lens[0]:])]

    def look(rows):
        q = rnd(2, h, d)
        out = c.attend(q, window=window, sinks=sinks)
        for b, (k, v) in enumerate(rows):
            ref, _, _, a, f = _attend(q[b], k, v, d ** -0.5, _visible(lens[b], window, sinks, "cuda"))
            _check_out(out[b], ref, a, f, lens[b], dt)

    for b in range(2):
        c.reserve(b, 100)
    rows = fill()
    look(rows)
    with pytest.raises(RuntimeError, match="budget"):
        c.evict(4, sinks=3, recent=2)                 # refused
    look(rows)
    c.evict(60, sinks=2, recent=5)                    # every row is within it
    look(rows)
    c.evict(30, sinks=2, recent=5)                    # cuts row 0
    with pytest.raises(RuntimeError, match="window"):
        c.attend(rnd(2, h, d), window=window)
    c.attend(rnd(2, h, d))
    c.release(1)                                      # was not cut
    with pytest.raises(RuntimeError, match="window"):
        c.attend(rnd(2, h, d), window=window)
    c.release(0)
    for b in range(2):
        c.reserve(b, 100)
    rows = fill()
    look(rows)
    # a captured eviction may be replayed at any time
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.evict(30, sinks=2, recent=5)
    look(rows)
    graph.replay()
    with pytest.raises(RuntimeError, match="window"):
        c.attend(rnd(2, h, d), window=window)
    for b in range(2):
        c.release(b)
        c.reserve(b, 100)
    rows = fill()
    look(rows)
    graph.replay()
    with pytest.raises(RuntimeError, match="window"):
        c.attend(rnd(2, h, d), window=window)
    ops.check_status(c.lens.device)


# ---------------------------------------------------------------------------------------
# evictions: many rows, lengths written over what the call reads
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("d, budget", [(8, 3), (8, 200), (5, 3)])
def test_evict_of_very_many_rows(d, budget):
    from project_chronos_b200 import ops
    b, g, n = 70000, 1, 4
    size = 4
    kp = torch.randn(b, size, g, d, generator=_gen(1), device="cuda").to(BF)
    vp = torch.randn(b, size, g, d, generator=_gen(2), device="cuda").to(BF)
    table = torch.randperm(b, generator=_gen(3), device="cuda").to(torch.int32).view(b, 1)
    w = torch.rand(b, g, size, generator=_gen(4), device="cuda")
    pos = torch.arange(size, dtype=torch.int32, device="cuda").expand(b, g, size).contiguous()
    ln = torch.full((b,), n, dtype=torch.int32, device="cuda")
    k0, v0 = kp[table[:, 0].long()].clone(), vp[table[:, 0].long()].clone()
    r = ops.paged_evict(kp, vp, table, ln, ln, w.clone(), pos, budget)
    ops.check_status(kp.device)
    m = min(n, budget)
    assert bool((r["lens"] == m).all()) and r["src"].shape == (b, g, budget)
    src = torch.arange(m, device="cuda").expand(b, m).clone()
    if budget < n:                                    # the smallest goes, the last slot fills its place
        low = w[:, 0].argmin(dim=1)
        gone = low < m
        src[gone, low[gone]] = n - 1
    assert torch.equal(r["src"][:, 0, :m].long(), src)
    at = src[:, :, None].expand(b, m, d)
    assert torch.equal(kp[table[:, 0].long()][:, :m, 0], k0[:, :, 0].gather(1, at))
    assert torch.equal(vp[table[:, 0].long()][:, :m, 0], v0[:, :, 0].gather(1, at))


@gpu
@pytest.mark.parametrize("lens_is", ["seen", "lens"])
def test_evict_writes_lengths_over_its_inputs(lens_is):
    """One slot too many in rows of many kv heads: the new lengths may take the place of what the call reads."""
    from project_chronos_b200 import ops
    lens, g, d, budget = [65] * 30 + [40, 64], 16, 16, 64
    kp, vp, table, ln, _ = _make_cache(lens, g, d, 16, BF, seed=1, bad=0.0)
    cap = table.shape[1] * 16
    w = torch.rand(len(lens), g, cap, generator=_gen(2), device="cuda")
    pos = torch.arange(cap, dtype=torch.int32, device="cuda").expand(len(lens), g, cap).contiguous()
    seen = ln.clone()
    ref = ops.paged_evict(kp.clone(), vp.clone(), table, ln, seen, w.clone(), pos.clone(), budget, sinks=2, recent=9)
    k, v = kp.clone(), vp.clone()
    r = ops.paged_evict(k, v, table, ln, seen, w, pos, budget, sinks=2, recent=9, lens_out=seen if lens_is == "seen" else ln)
    for key in ("lens", "src", "weights", "positions"):
        assert torch.equal(r[key], ref[key])


# ---------------------------------------------------------------------------------------
# prompts: expanded heads, results over the queries, offsets
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("which", ["q", "k", "v", "k and v", "all"])
@pytest.mark.parametrize("dt", [BF, FP])
def test_prompt_attention_takes_expanded_heads(which, dt):
    """One row of heads read as several: strides of zero."""
    from project_chronos_b200 import ops
    n, h, g, d = 300, 8, 4, 64
    gen = _gen(4)
    make = lambda heads, name: torch.randn(n, 1 if name in which or which == "all" else heads, d, generator=gen,  # noqa: E731
                                           device="cuda").to(dt).expand(n, heads, d)
    q, k, v = make(h, "q"), make(g, "k"), make(g, "v")
    cu = torch.tensor([0, 100, n], dtype=torch.int32, device="cuda")
    out = ops.window_attention(q, k, v, cu, window=90, sinks=2)
    for c0, m in ((0, 100), (100, 200)):
        _check_prompt(out, None, q, k, v, m, m, c0, c0, 90, 2, dt, _some_rows(m))


@gpu
@pytest.mark.parametrize("lq, lk", [(300, 300), (40, 4000)])
@pytest.mark.parametrize("bad", [False, True])
def test_prompt_attention_over_its_queries(lq, lk, bad):
    """out may be q, also where a value that is not finite sends rows through a second computation."""
    from project_chronos_b200 import ops
    h, g, d, window = 8, 2, 128, 200
    gen = _gen(1)
    q, k, v = (torch.randn(r, x, d, generator=gen, device="cuda").to(BF) for r, x in ((lq, h), (lk, g), (lk, g)))
    if bad:
        v[lk - 20, :, 3] = math.inf
    cq, ck = (torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (lq, lk))
    want = ops.window_attention(q, k, v, cq, cu_seqlens_k=ck, window=window)
    got = q.clone()
    ops.window_attention(got, k, v, cq, cu_seqlens_k=ck, window=window, out=got)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_offsets_that_do_not_ascend_are_reported(dt):
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    q, k = torch.zeros(9, 4, 64, dtype=dt, device="cuda"), torch.zeros(9, 2, 64, dtype=dt, device="cuda")
    for cu in ([0, 9, 3], [0, 4, 4, 9, 2], list(range(9)) + [9] * 60 + [5], [9, 3], [3, 2, 1, 0]):
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        ops.window_attention(q, k, k, cu)
        with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
            ops.check_status(q.device)


@gpu
def test_sums_that_require_grad_are_refused():
    from project_chronos_b200 import ops
    kp, vp, table, ln, _ = _make_cache([5, 6], 2, 64, 16, BF, seed=1)
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    w = torch.zeros(2, 2, 32, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.paged_attn_decode(q, kp, vp, table, ln, weights=w)
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.paged_attn_decode(q, kp, vp, table, ln, lse=torch.zeros(2, 4, device="cuda", requires_grad=True))
    with torch.no_grad():
        ops.paged_attn_decode(q, kp, vp, table, ln, weights=w)


def test_trim_refuses_negative_slots():
    from project_chronos_b200 import PagedCache
    c = PagedCache(1, 5, 1, 8, 4, "cpu", torch.float32, page_size=4)
    c.reserve(0, 12)
    for call in (c.trim, c.reserve):
        with pytest.raises(ValueError, match="negative"):
            call(0, -5)
    assert c.page_table.tolist() == [[0, 1, 2, -1]] and c.free_pages() == 2


def test_trim_cuts_the_length():
    """Slots whose pages were given back do not come back with other pages."""
    from project_chronos_b200 import PagedCache
    c = PagedCache(2, 8, 1, 8, 4, "cpu", torch.float32, page_size=4)
    for row, slots in ((0, 14), (1, 6)):
        c.reserve(row, slots)
        c.lens[row], c.seen[row] = slots, slots
    c.trim(0, 5)
    assert c.lens.tolist() == [8, 6] and c.seen.tolist() == [14, 6]
    c.reserve(0, 16)
    assert c.lens.tolist() == [8, 6]
    c.trim(1, 8)                                      # nothing behind it
    assert c.lens.tolist() == [8, 6]


def test_results_that_overlap_other_inputs_are_refused(lib):
    from project_chronos_b200 import _native as N
    cap = 8                                           # 2 * 2 * 8 numbers
    for at in (4096 - 4, 4096 + 4, 4096 + 127):
        d = N.ChronosPagedDecodeArgs(cache=_native_cache(N), heads=4, scale=1.0, weights=4096, weights_out=at, slot_cap=cap)
        assert lib.chronos_paged_decode(ctypes.byref(d), None) == N.CHRONOS_ERR_INVALID_ARG
        assert b"overlaps" in lib.chronos_moe_last_error()
        for f in (dict(weights_out=at, positions_out=8192), dict(weights_out=4096, positions_out=at + 4096)):
            e = N.ChronosPagedEvictArgs(cache=_native_cache(N), budget=4, weights=4096, positions=8192, slot_cap=cap, **f)
            assert lib.chronos_paged_evict(ctypes.byref(e), None) == N.CHRONOS_ERR_INVALID_ARG
            assert b"overlap" in lib.chronos_moe_last_error()
    for at in (4096, 4096 + 128, 4096 - 128):         # the same, side by side
        d = N.ChronosPagedDecodeArgs(cache=_native_cache(N), heads=4, scale=1.0, weights=4096, weights_out=at, slot_cap=cap)
        assert lib.chronos_paged_decode(ctypes.byref(d), None) == N.CHRONOS_ERR_INVALID_ARG
        assert b"required" in lib.chronos_moe_last_error()
    for f in (dict(k=4096, v=8192), dict(k=8192, v=4096)):
        w = N.ChronosWindowAttnArgs(batch=1, heads=2, kv_heads=2, head_dim=8, scale=1.0, num_q=4, num_k=4, q=1024, out=4096,
                                    cu_q=512, cu_k=512, **f)
        assert lib.chronos_window_attention(ctypes.byref(w), None) == N.CHRONOS_ERR_INVALID_ARG
        assert b"not k or v" in lib.chronos_moe_last_error()


@gpu
@pytest.mark.parametrize("packed", [False, True])
def test_a_captured_step_counts_what_it_stored(packed):
    """Append and attention in one graph, replayed while a row grows, fills up and gets more pages."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import PagedCache, ops
    h, g, d, dt = 8, 2, 64, BF
    c = PagedCache(2, 12, g, d, 6, "cuda", dt, page_size=16, track_weights=True)
    k, v = (torch.zeros(2, g, d, dtype=dt, device="cuda") for _ in range(2))
    q, out = torch.zeros(2, h, d, dtype=dt, device="cuda"), torch.zeros(2, h, d, dtype=dt, device="cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda") if packed else None
    for b in range(2):
        c.reserve(b, 16 + 32 * b)

    def step():
        c.append(k, v, cu)
        c.attend(q, out=out)

    step()                                            # a first call outside the capture
    for b in range(2):
        c.release(b)
        c.reserve(b, 16 + 32 * b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert c.lens.tolist() == [0, 0]                  # captured, not run
    book = [[], []]
    gen = _gen(3)
    for i in range(40):
        if i == 20:
            c.reserve(0, 40)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        graph.replay()
        full = 16 <= i < 20
        for b in range(2):
            if b == 1 or not full:
                book[b].append((k[b].clone(), v[b].clone()))
            ks, vs = (torch.stack([r[j] for r in book[b]]) for j in (0, 1))
            ref, _, _, a, f = _attend(q[b], ks, vs, d ** -0.5, _visible(len(ks), 0, 0, "cuda"))
            _check_out(out[b], ref, a, f, len(ks), dt)
        assert c.lens.tolist() == [len(x) for x in book] == c.seen.tolist()
        if full:
            with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
                ops.check_status(out.device)
        else:
            ops.check_status(out.device)
