"""The paged cache's further operators (include/chronos_paged4.h): append with rotation,
pages of 4-bit values, one-token attention over them, rows read back, page bounds,
selected pages and the attention over them.

CPU: refusals and bookkeeping.  GPU: every operator against its definition in 64 bits.
Tolerances, with u = finfo(type).eps / 2:

* a rotated column y = x c - x' s is two products and a sum in fp32, each off by at most
  2^-24 of its magnitude: 2^-23 (|x c| + |x' s|) in all; stored in 16 bits it is off by
  u |y| more (and by half the smallest step of fp16, 2^-25);
* codes, scales, copies, bounds, selected pages: equal, bit by bit;
* attention, with A = sum_j p_j |v_j|, S = max_j scale sum_d |q_d k_jd| and
  f = D 2^-23 S + n 2^-24 + 2^-20 as for the 16-bit cache: over 4-bit pages queries and
  weights are halves.  A query column is a half in units of a power of two of its head,
  the largest between 2^8 and 2^9: exact, but for columns so small that they are off by
  2^-25 of a unit, 2^-33 of the largest column q^: f grows by 2^-33 scale q^ sum_d |k_jd|
  <= 2^-33 sqrt(D) scale |q| |k| <= 2^-28 S' with S' = scale |q| max_j |k_j| (D <= 256);
  fp32 layers split columns and weights into two halves, off by 2^-22: f grows by
  2^-21 S + 2^-22.  Weights of 16-bit layers are off by 2^-11 A, those of all by 2^-25
  in units of 2^-7 of the heaviest or more: n 2^-32 max |v|;
  the result is rounded once (u |out|).
"""
import ctypes
import math

import pytest
import torch

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _unit(dt):
    return torch.finfo(dt).eps / 2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(seed, *shape, dt=FP, scale=1.0):
    return (scale * torch.randn(shape, generator=_gen(seed), device="cuda")).to(dt)


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------
# no GPU: refusals, sizes, bookkeeping
# ---------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def lib():
    from project_chronos_b200 import _native, build
    build.build()
    return _native.load_library()


def _native_cache(N, **kw):
    f = dict(batch=2, kv_heads=2, head_dim=16, dtype=N.DTYPE_BF16, num_pages=4, page_size=16, table_width=2)
    f.update(kw)
    return N.ChronosPagedCache(**f)


def test_cpu_tensors_are_refused():
    from project_chronos_b200 import ops
    k = torch.zeros(2, 2, 16)
    q = torch.zeros(2, 4, 16)
    kp, table, lens = torch.zeros(4, 4, 2, 16), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    p4 = torch.zeros(4, 2, ops.packed_page_bytes(16, 16), dtype=torch.uint8)
    bounds = torch.zeros(4, 2, 2, 16)
    for call in (lambda: ops.paged_append_rope(k, k, kp, kp, table, lens), lambda: ops.paged_attn_decode4(q, p4, p4, table, lens),
                 lambda: ops.paged_gather(kp, kp, table, lens, lens, k, k), lambda: ops.paged_bounds(kp, bounds, table, lens),
                 lambda: ops.paged_select(q, bounds, table, lens, 4, 2),
                 lambda: ops.paged_attn_sparse(q, kp, kp, table, lens, torch.zeros(2, 2, 2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("d, columns", [(1, 64), (64, 64), (65, 128), (96, 128), (128, 128), (129, 256), (256, 256)])
def test_packed_sizes(d, columns):
    from project_chronos_b200 import ops
    assert ops.packed_columns(d) == columns
    assert ops.packed_page_bytes(48, d) == 48 * columns * 9 // 16
    for bad in (0, 8, 40, -16):
        with pytest.raises(ValueError, match="multiple of 16"):
            ops.packed_page_bytes(bad, d)
    for bad in (0, 257):
        with pytest.raises(ValueError, match="head_dim"):
            ops.packed_columns(bad)


def _refuses(lib, name, args, text, workspace=False):
    from project_chronos_b200 import _native as N
    assert getattr(lib, "chronos_paged_" + name)(ctypes.byref(args), None) == N.CHRONOS_ERR_INVALID_ARG
    assert text in lib.chronos_moe_last_error()
    if workspace:
        assert getattr(lib, f"chronos_paged_{name}_workspace")(ctypes.byref(args)) == 0


@pytest.mark.parametrize("change, text", [
    (dict(cache=dict(head_dim=257)), b"head_dim"), (dict(cache=dict(dtype=9)), b"dtype"), (dict(num_tokens=-1), b"num_tokens"),
    (dict(num_tokens=3), b"cu_seqlens"), (dict(heads=-1), b"heads"), (dict(rope_dim=3), b"rotation"), (dict(rope_dim=-2), b"rotation"),
    (dict(rope_dim=16, rope_start=2), b"rotation"), (dict(rope_start=-1), b"rotation"),
    (dict(rope_dim=4, table_dtype=9), b"table_dtype"), (dict(rope_dim=4, table_len=-1), b"table_len"),
    (dict(rope_dim=4, table_dtype=0), b"seen"), (dict(positions=256), b"seen"), (dict(seen_out=256), b"seen"),
    (dict(weights=256, slot_cap=-1), b"slot_cap"), (dict(lens_out=256, seen_out=256, seen=4096), b"overlap"),
    (dict(q=512, q_out=512, heads=2, q_row_stride=8), b"same strides"), (dict(k=512, k_out=512, k_row_stride=8), b"same strides"),
    (dict(k=512, k_out=520, k_row_stride=64, k_out_row_stride=64), b"overlap"), (dict(v=512, k_out=512), b"overlap"),
    (dict(packed=1, k_scale=0.0, v_scale=1.0), b"k_scale"), (dict(packed=1, k_scale=1.0, v_scale=float("nan")), b"v_scale"),
    (dict(packed=1, k_scale=1.0, v_scale=1.0, cache=dict(page_size=8)), b"page_size"),
    (dict(packed=1, k_scale=1.0, v_scale=1.0, cache=dict(k_page_stride=24)), b"multiples of 16"), ({}, b"required"),
])
def test_append_rope_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(num_tokens=2)
    f.update({k: v for k, v in change.items() if k != "cache"})
    _refuses(lib, "append_rope", N.ChronosPagedRopeArgs(cache=_native_cache(N, **change.get("cache", {})), **f), text)


@pytest.mark.parametrize("change, text", [
    (dict(heads=3), b"heads"), (dict(heads=0), b"heads"), (dict(heads=2 * 257), b"heads"), (dict(window=-1), b"window"),
    (dict(sinks=-1), b"sinks"), (dict(scale=0.0), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(k_scale=-1.0), b"k_scale"),
    (dict(v_scale=0.0), b"v_scale"), (dict(cache=dict(page_size=24)), b"page_size"), (dict(cache=dict(v_head_stride=8)), b"multiples of 16"),
    (dict(cache=dict(batch=-1)), b"batch"), ({}, b"required"),
])
def test_decode4_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(heads=4, scale=0.25, k_scale=1.0, v_scale=1.0)
    f.update({k: v for k, v in change.items() if k != "cache"})
    a = N.ChronosPagedDecode4Args(cache=_native_cache(N, **change.get("cache", {})), **f)
    _refuses(lib, "decode4", a, text, workspace=bool(change))


@pytest.mark.parametrize("change, text", [
    (dict(topk=2, first=1, last=2), b"topk"), (dict(last=0), b"topk"), (dict(first=-1), b"topk"), (dict(heads=5), b"heads"),
    (dict(num_tokens=5), b"cu_seqlens"), (dict(num_tokens=-1), b"num_tokens"), (dict(cache=dict(page_size=0)), b"page_size"), ({}, b"required"),
])
def test_select_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(heads=4, topk=4, first=0, last=1, num_tokens=2)
    f.update({k: v for k, v in change.items() if k != "cache"})
    _refuses(lib, "select", N.ChronosPagedSelectArgs(cache=_native_cache(N, **change.get("cache", {})), **f), text)


@pytest.mark.parametrize("change, text", [
    (dict(topk=-1), b"topk"), (dict(topk=1 << 27), b"topk"), (dict(heads=5), b"heads"), (dict(scale=-1.0), b"scale"),
    (dict(num_tokens=5), b"cu_seqlens"), (dict(packed=1, k_scale=0.0), b"k_scale"), ({}, b"required"),
])
def test_sparse_refuses_before_touching_the_device(lib, change, text):
    from project_chronos_b200 import _native as N
    f = dict(heads=4, topk=2, scale=1.0, k_scale=1.0, v_scale=1.0, num_tokens=2)
    f.update(change)
    _refuses(lib, "sparse", N.ChronosPagedSparseArgs(cache=_native_cache(N), **f), text)


def test_gather_and_bounds_refuse_before_touching_the_device(lib):
    from project_chronos_b200 import _native as N
    _refuses(lib, "gather", N.ChronosPagedGatherArgs(cache=_native_cache(N), num_tokens=-1), b"num_tokens")
    _refuses(lib, "gather", N.ChronosPagedGatherArgs(cache=_native_cache(N), num_tokens=1), b"required")
    _refuses(lib, "gather", N.ChronosPagedGatherArgs(cache=_native_cache(N), num_tokens=1, packed=1), b"k_scale")
    _refuses(lib, "bounds", N.ChronosPagedBoundsArgs(cache=_native_cache(N), num_tokens=-1), b"num_tokens")
    _refuses(lib, "bounds", N.ChronosPagedBoundsArgs(cache=_native_cache(N)), b"required")
    _refuses(lib, "bounds", N.ChronosPagedBoundsArgs(cache=_native_cache(N, page_size=8), packed=1, k_scale=1.0), b"page_size")


def test_empty_calls_return_without_a_device(lib):
    from project_chronos_b200 import _native as N
    c = _native_cache(N, batch=0)
    one = dict(k_scale=1.0, v_scale=1.0)
    for name, a in (("append_rope", N.ChronosPagedRopeArgs(cache=c)), ("gather", N.ChronosPagedGatherArgs(cache=c)),
                    ("decode4", N.ChronosPagedDecode4Args(cache=c, heads=2, scale=1.0, **one)),
                    ("bounds", N.ChronosPagedBoundsArgs(cache=c)), ("select", N.ChronosPagedSelectArgs(cache=c, heads=2, topk=1, last=1)),
                    ("sparse", N.ChronosPagedSparseArgs(cache=c, heads=2, scale=1.0, **one))):
        assert getattr(lib, "chronos_paged_" + name)(ctypes.byref(a), None) == N.CHRONOS_OK, name


def test_select_workspace_is_bounded(lib):
    from project_chronos_b200 import _native as N
    def need(width, topk, tokens):
        a = N.ChronosPagedSelectArgs(cache=_native_cache(N, batch=tokens, table_width=width), heads=2, topk=topk, last=1, num_tokens=tokens)
        return lib.chronos_paged_select_workspace(ctypes.byref(a))
    assert need(8, 8, 4) == 0                          # every row takes all it has
    assert need(9, 8, 4) == 4 * 2 * 9 * 8
    assert need(1 << 15, 8, 1 << 14) <= 1 << 28
    assert need(1 << 26, 8, 2) == 2 * 8 << 26          # one token's, where those are more


def test_cache_kinds_on_the_host():
    from project_chronos_b200 import PagedCache, ops
    c = PagedCache(2, 5, 3, 80, 4, "cpu", BF, page_size=32, four_bit=True, page_bounds=True)
    assert c.k_pages.dtype == torch.uint8 and c.k_pages.shape == (5, 3, ops.packed_page_bytes(32, 80))
    assert c.bounds.shape == (5, 2, 3, 80) and c.bounds.dtype == BF
    assert c.nbytes() == 2 * c.k_pages.numel() + 2 * c.bounds.numel()
    c.reserve(0, 33)
    assert c.page_table.tolist()[0][:2] == [0, 1]
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(3)
    for kind in (dict(four_bit=True), dict(page_bounds=True)):
        with pytest.raises(ValueError, match="track_weights"):
            PagedCache(2, 5, 3, 80, 4, "cpu", BF, page_size=32, track_weights=True, **kind)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCache(2, 5, 3, 80, 4, "cpu", BF, page_size=8, four_bit=True)
    with pytest.raises(RuntimeError, match="page_bounds"):
        PagedCache(2, 5, 3, 80, 4, "cpu", BF).attend_sparse(torch.zeros(2, 3, 80), 2)


# ---------------------------------------------------------------------------------------
# definitions
# ---------------------------------------------------------------------------------------

def _rotate(x, cos, sin, start):
    """x [T, heads, D] in 64 bits, cos and sin [T, R]: (rotated, what each column's magnitudes add up to)."""
    r = cos.shape[1]
    y, m = x.clone(), x.abs()
    a, b = x[..., start: start + r // 2], x[..., start + r // 2: start + r]
    c, s = cos[:, None].double(), sin[:, None].double()
    h = r // 2
    y[..., start: start + h] = a * c[..., :h] - b * s[..., :h]
    y[..., start + h: start + r] = b * c[..., h:] + a * s[..., h:]
    m[..., start: start + h] = (a * c[..., :h]).abs() + (b * s[..., :h]).abs()
    m[..., start + h: start + r] = (b * c[..., h:]).abs() + (a * s[..., h:]).abs()
    return y, m


def _near(got, y, m, dt):
    tol = 2.0 ** -23 * m + (0.0 if dt == FP else _unit(dt)) * y.abs() + (2.0 ** -25 if dt == HF else 0.0) + (2.0 ** -24 * y.abs() if dt == FP else 0.0)
    err = (got.double() - y).abs()
    assert bool((err <= tol * 1.001 + 1e-40).all()), float((err / (tol + 1e-40)).max())


def _quantise(x, unit=1.0):
    """Rows x [..., D] in 64 bits as the pages hold them: codes [..., D], scale bytes [..., blocks] and the values.
    Level by level, from the definition."""
    d = x.shape[-1]
    y = torch.nn.functional.pad(x, (0, -d % 16)).unflatten(-1, (-1, 16)) / torch.tensor(unit, dtype=torch.float32, device=x.device).double()
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    top = (y.abs().amax(-1) / 6).float().clamp(max=448.0)
    scale = top.to(torch.float8_e4m3fn)
    s = scale.double()[..., None]
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    code = torch.zeros(y.shape, dtype=torch.int64, device=x.device)
    for i in range(7):
        edge = (lv[i] + lv[i + 1]) / 2 * s             # exact
        code = torch.where((y.abs() > edge) | ((y.abs() == edge) & (i % 2 == 1)), i + 1, code)
    code = torch.where(s == 0, 0, code + 8 * torch.signbit(y).long())
    scales = torch.where(bad, 127, scale.view(torch.uint8).long())
    sign = torch.where(code >= 8, -1.0, 1.0)
    value = sign * lv[code % 8] * s * float(torch.tensor(unit, dtype=torch.float32))
    value = torch.where(bad[..., None], math.nan, value)
    return code.flatten(-2)[..., :d], scales, value.flatten(-2)[..., :d]


def _stored(pages, table, d, size, slots):
    """Codes, scale bytes and values of a sequence's slots: pages [n, G, bytes], its table row -> [slots, G, ...]."""
    from project_chronos_b200 import ops
    p = ops.packed_columns(d)
    record = pages.view(pages.shape[0], pages.shape[1], size // 16, 9 * p)[table.long()[slots // size], :, slots % size // 16]   # [n, G, 9P]
    line = slots % 16
    at = torch.arange(slots.shape[0], device=pages.device)
    b = record[..., : 8 * p].unflatten(-1, (16, p // 2))[at, :, line].long()
    code = torch.stack([b % 16, b // 16], dim=-1).flatten(-2)
    scale = record[..., 8 * p:].unflatten(-1, (16, p // 16))[at, :, line]
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=pages.device)
    value = torch.where(code >= 8, -1.0, 1.0) * lv[code % 8] * scale.contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, dim=-1)
    return code, scale.long(), value[..., :d]


def _tables(n, r, dt=FP, base=1e4):
    f = base ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / max(r, 1))
    a = torch.outer(torch.arange(n, device="cuda", dtype=torch.float64), f)
    return torch.cat([a.cos(), a.cos()], 1).to(dt), torch.cat([a.sin(), a.sin()], 1).to(dt)


def _page_table(b, width, spare, seed):
    n = b * width + spare
    return torch.randperm(n, generator=_gen(seed), device="cuda")[: b * width].view(b, width).to(torch.int32).contiguous(), n


def _attend(q, k, v, scale):
    """q [H, D], k and v [n, G, D] in 64 bits: out, lse, A, S, S'."""
    h, g = q.shape[0], k.shape[1]
    k, v, q = k.double().repeat_interleave(h // g, 1), v.double().repeat_interleave(h // g, 1), q.double()
    x = torch.einsum("hd,nhd->hn", q, k) * scale
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None]) if k.shape[0] else x
    out, a = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
    if k.shape[0] == 0:
        z = torch.zeros(h, dtype=torch.float64, device=q.device)
        return out, lse, a, z, z
    s = (torch.einsum("hd,nhd->hn", q.abs(), k.abs()) * scale).amax(1)
    return out, lse, a, s, q.norm(dim=1) * k.norm(dim=2).amax(0) * scale


def _check_attention(out, lse, q, k, v, scale, dt, four):
    n, d = k.shape[0], q.shape[1]
    ref, rl, a, s, s2 = _attend(q, k, v, scale)
    f = d * 2.0 ** -23 * s + n * 2.0 ** -24 + 2.0 ** -20
    vmax = v.double().abs().max() if n else 0.0
    if four:
        f = f + 2.0 ** -28 * s2 + (2.0 ** -21 * s + 2.0 ** -22 if dt == FP else 0.0)
        weights = 2.0 ** -11 if dt != FP else 0.0
        floor = n * 2.0 ** -32 * vmax
    else:
        weights = _unit(dt) if dt != FP else 0.0
        floor = 2.0 ** -25 * n * vmax if dt == HF else 0.0
    tol = _unit(dt) * ref.abs() + (f[:, None] + n * 2.0 ** -23 + weights) * a + floor + (2.0 ** -25 if dt == HF else 0.0) + 1e-30
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the tolerance"
    if lse is not None:
        if n == 0:
            assert bool((lse == -math.inf).all())
        else:
            assert bool(((lse.double() - rl).abs() <= f + 2.0 ** -22 * rl.abs()).all())


# ---------------------------------------------------------------------------------------
# append with rotation, layer-type pages
# ---------------------------------------------------------------------------------------

def _layout(kind, t, heads, d, dt, seed):
    """Rows [t, heads, d] laid out densely, as a part of wider rows, or so that no vector loads fit."""
    if kind == "dense":
        return _rnd(seed, t, heads, d, dt=dt)
    if kind == "wide":
        return _rnd(seed, t, heads + 3, d, dt=dt)[:, 2: 2 + heads]
    return _rnd(seed, t, heads, d + 1, dt=dt)[..., 1:]


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d, r, start, size", [(8, 2, 128, 128, 0, 16), (4, 4, 64, 32, 32, 64), (10, 2, 80, 80, 0, 48), (6, 1, 96, 48, 0, 32),
                                                     (16, 2, 256, 64, 192, 16), (3, 3, 37, 10, 5, 7), (1, 1, 1, 0, 0, 1), (0, 5, 40, 2, 38, 3)])
@pytest.mark.parametrize("new", [None, [1, 0, 40, 3], [17, 1, 1, 200]])
@pytest.mark.parametrize("layout", ["dense", "wide", "odd"])
def test_append_rope_matches_its_definition(dt, h, g, d, r, start, size, new, layout):
    from project_chronos_b200 import ops
    before, seen = [0, 15, 64, 7], [3, 15, 70, 7]
    b, lens = 4, new or [1] * 4
    t, pad = sum(lens), 0 if new is None else 2
    width = -(-max(x + n for x, n in zip(before, lens)) // size)
    table, n = _page_table(b, width, 2, 1)
    kp, vp = _rnd(2, n, size, g, d, dt=dt), _rnd(3, n, size, g, d, dt=dt)
    k0, v0 = kp.clone(), vp.clone()
    k, v = _layout(layout, t + pad, g, d, dt, 4), _layout(layout, t + pad, g, d, dt, 5)
    q = _layout(layout, t + pad, h, d, dt, 6) if h else None
    tt = dt if size == 16 else FP
    cos, sin = _tables(max(s + n for s, n in zip(seen, lens)), r, tt)
    cap = width * size
    w, pos = torch.full((b, g, cap), 5.0, device="cuda"), torch.full((b, g, cap), 9, dtype=torch.int32, device="cuda")
    cu = None if new is None else torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    ln, sn = _i32(*before), _i32(*seen)
    q_out = torch.full((t + pad, max(h, 1), d), 7.0, dtype=dt, device="cuda")
    k_out = torch.full((t + pad, g, d), 7.0, dtype=dt, device="cuda")
    res = ops.paged_append_rope(k, v, kp, vp, table, ln, sn, cos if r else None, sin if r else None, q=q, q_out=q_out if h else None,
                                k_out=k_out, cu_seqlens=cu, rope_start=start, weights=w, positions=pos, lens_out=ln, seen_out=sn)
    ops.check_status(kp.device)
    assert (res is None) == (h == 0) and (res is None or res is q_out)
    assert ln.tolist() == [x + n for x, n in zip(before, lens)] and sn.tolist() == [x + n for x, n in zip(seen, lens)]
    at = 0
    for i in range(b):
        m = lens[i]
        rows, slots = slice(at, at + m), torch.arange(before[i], before[i] + m, device="cuda")
        c, s = cos[seen[i]: seen[i] + m], sin[seen[i]: seen[i] + m]
        y, mag = _rotate(k[rows].double(), c, s, start)
        to = table[i].long()[slots // size], slots % size
        _near(kp[to], y, mag, dt)
        assert torch.equal(kp[to], k_out[rows])
        assert torch.equal(vp[to], v[rows])
        if h:
            _near(q_out[rows], *_rotate(q[rows].double(), c, s, start), dt)
        k0[to], v0[to] = kp[to], vp[to]
        live = torch.zeros(cap, dtype=torch.bool, device="cuda")
        live[slots] = True
        assert bool((w[i] == torch.where(live, 0.0, 5.0)).all())
        assert torch.equal(pos[i][:, slots], torch.arange(seen[i], seen[i] + m, device="cuda", dtype=torch.int32).expand(g, m))
        assert bool((pos[i][:, ~live] == 9).all())
        at += m
    assert torch.equal(kp, k0) and torch.equal(vp, v0)     # nothing else was written
    if pad:
        assert bool((q_out[t:] == 7.0).all()) and bool((k_out[t:] == 7.0).all())


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("d", [128, 37])
def test_append_rope_in_place(dt, d):
    """q_out may be q, k_out may be k (views of one projection)."""
    from project_chronos_b200 import ops
    h, g, t, size = 8, 2, 300, 16
    r = d // 2 * 2
    table, n = _page_table(2, 20, 0, 1)
    cu, zero = _i32(0, 100, 300), _i32(0, 0)
    cos, sin = _tables(200, r)
    qkv = _rnd(4, t, h + 2 * g, d, dt=dt)
    kp, vp = (torch.zeros(n, size, g, d, dtype=dt, device="cuda") for _ in range(2))
    k2, v2 = kp.clone(), vp.clone()
    q, k, v = qkv.clone().split([h, g, g], dim=1)
    want_k = torch.empty_like(k)
    want = ops.paged_append_rope(k, v, kp, vp, table, zero, zero, cos, sin, q=q, k_out=want_k, cu_seqlens=cu)
    q, k, v = qkv.split([h, g, g], dim=1)
    got = ops.paged_append_rope(k, v, k2, v2, table, zero, zero, cos, sin, q=q, q_out=q, k_out=k, cu_seqlens=cu)
    assert got is q and torch.equal(q, want) and torch.equal(k, want_k) and torch.equal(kp, k2) and torch.equal(vp, v2)
    for bad in (dict(q=q, q_out=qkv[:, 1: h + 1]), dict(k_out=v), dict(q=q, q_out=qkv[:, g: g + h]), dict(q=q, q_out=q, k_out=q[:, :g])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.paged_append_rope(k, v, k2, v2, table, zero, zero, cos, sin, cu_seqlens=cu, **bad)
    # heads in turn: query, key and value of a head side by side
    each = _rnd(5, t, g, 3, d, dt=dt)
    q, k, v = (x.clone() for x in each.unbind(2))
    want = ops.paged_append_rope(k, v, kp, vp, table, zero, zero, cos, sin, q=q, cu_seqlens=cu)
    q, k, v = each.unbind(2)
    ops.paged_append_rope(k, v, k2, v2, table, zero, zero, cos, sin, q=q, q_out=q, k_out=k, cu_seqlens=cu)
    assert torch.equal(q, want) and torch.equal(kp, k2) and torch.equal(vp, v2)


@gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("four", [False, True])
def test_append_rope_drops_what_has_no_place(packed, four):
    """A position behind the tables, a slot behind the pages, a page that is none: dropped, reported, not counted."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    h, g, d, size, dt = 4, 2, 64, 16, BF
    new = [3, 4, 2, 5] if packed else [1] * 4
    before = [30, 15, 0, 2]                                # of 32 slots
    seen = [4, 98, 0, 2]
    table = _i32(*[0, 1, 2, 3, 99, 5, 6, 7]).view(4, 2)    # row 2's first page is none
    t = sum(new)
    cos, sin = _tables(100, d)                             # row 1's tokens from its third on lie behind them
    if not packed:
        before[0], seen[1] = 32, 100
    cu = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32) if packed else None
    if four:
        kp, vp = (torch.full((8, g, ops.packed_page_bytes(size, d)), 9, dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        kp, vp = (torch.full((8, size, g, d), 9.0, dtype=dt, device="cuda") for _ in range(2))
    ln, sn = _i32(*before), _i32(*seen)
    q, k, v = (_rnd(i, t, x, d, dt=dt) for i, x in ((1, h), (2, g), (3, g)))
    k_out = torch.empty_like(k)
    got = ops.paged_append_rope(k, v, kp, vp, table, ln, sn, cos, sin, q=q, k_out=k_out, cu_seqlens=cu, lens_out=ln, seen_out=sn)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(kp.device)
    stored = [2, 2, 0, 5] if packed else [0, 0, 0, 1]
    assert ln.tolist() == [x + n for x, n in zip(before, stored)] and sn.tolist() == [x + n for x, n in zip(seen, stored)]
    at = 0
    for i, n in enumerate(new):
        for j in range(n):
            p = seen[i] + j
            if p >= 100:
                assert not bool(got[at].any()) and not bool(k_out[at].any())
            else:
                _near(got[at: at + 1], *_rotate(q[at: at + 1].double(), cos[p: p + 1], sin[p: p + 1], 0), dt)
                _near(k_out[at: at + 1], *_rotate(k[at: at + 1].double(), cos[p: p + 1], sin[p: p + 1], 0), dt)
            at += 1
    for x in (kp, vp):                                     # pages that nothing went into
        assert bool((x[4: 6] == 9).all())


@gpu
def test_append_rope_of_no_tokens():
    from project_chronos_b200 import ops
    kp = torch.ones(4, 16, 2, 64, dtype=BF, device="cuda")
    table, ln, sn = _i32(0, 1, 2, 3).view(2, 2), _i32(5, 6), _i32(7, 8)
    none = torch.empty(0, 2, 64, dtype=BF, device="cuda")
    q = ops.paged_append_rope(none, none, kp, kp.clone(), table, ln, sn, *_tables(9, 64), q=none, cu_seqlens=_i32(0, 0, 0),
                              lens_out=ln, seen_out=sn)
    assert q.shape == (0, 2, 64) and ln.tolist() == [5, 6] and sn.tolist() == [7, 8] and bool((kp == 1).all())
    ops.check_status(kp.device)


# ---------------------------------------------------------------------------------------
# 4-bit pages
# ---------------------------------------------------------------------------------------

def _values(t, g, d, dt, seed):
    """Rows with what quantisation meets: ordinary values, blocks of zeros, large and tiny ones, values on the borders
    between codes, alone among zeros, blocks that are not finite."""
    x = _rnd(seed, t, g, d)
    m = torch.arange(t, device="cuda") % 9
    lv = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device="cuda")
    border = lv[torch.randint(0, 8, (t, g, d), generator=_gen(seed + 1), device="cuda")] * torch.sign(x)
    border[..., ::16] = 6.0
    x = torch.where((m == 1)[:, None, None], 0.0, x)
    x = torch.where((m == 2)[:, None, None], x * 3e4 if dt == HF else x * 1e30, x)
    x = torch.where((m == 3)[:, None, None], x * 1e-3, x)
    x = torch.where((m == 4)[:, None, None], border * 0.3125, x)     # scale 0.3125 exactly
    x = torch.where(((m == 5)[:, None] & (torch.arange(g, device="cuda") % 2 == 0))[..., None] & (torch.arange(d, device="cuda") % 16 != 3), 0.0, x)
    x = torch.where((m == 6)[:, None, None], torch.exp(3 * x) * torch.sign(x), x)
    bad = (m == 7)[:, None, None] & (torch.arange(d, device="cuda") == d // 2)
    x = torch.where(bad, torch.where(torch.arange(g, device="cuda")[:, None] % 2 == 0, math.nan, -math.inf), x)
    return x.to(dt)


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("g, d, r, size", [(2, 128, 128, 16), (3, 64, 32, 64), (1, 80, 80, 48), (2, 96, 48, 32), (1, 256, 64, 16), (3, 37, 10, 16), (2, 1, 0, 16)])
@pytest.mark.parametrize("units", [(1.0, 1.0), (0.25, 16.0), (0.37, 3.1)])
def test_4bit_pages_hold_the_nearest_codes(dt, g, d, r, size, units):
    """Codes and scales are those of exact arithmetic, on borders too."""
    from project_chronos_b200 import ops
    new, before, seen = [1, 0, 180, 33], [0, 15, 64, 7], [3, 15, 70, 7]
    t = sum(new)
    width = -(-max(x + n for x, n in zip(before, new)) // size)
    table, n = _page_table(4, width, 2, 1)
    kp, vp = (torch.randint(0, 256, (n, g, ops.packed_page_bytes(size, d)), generator=_gen(i), device="cuda", dtype=torch.uint8) for i in (2, 3))
    k0, v0 = kp.clone(), vp.clone()
    k, v = _values(t, g, d, dt, 5), _values(t, g, d, dt, 8)
    cos, sin = _tables(300, r)
    cu = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    ln, sn = _i32(*before), _i32(*seen)
    ops.paged_append_rope(k, v, kp, vp, table, ln, sn, cos if r else None, sin if r else None, cu_seqlens=cu, k_scale=units[0], v_scale=units[1])
    ops.check_status(kp.device)
    k_out, v_out = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    after = ln + torch.tensor(new, dtype=torch.int32, device="cuda")
    ops.paged_gather(kp, vp, table, after, cu, k_out, v_out, k_scale=units[0], v_scale=units[1])
    ops.check_status(kp.device)
    at = 0
    p = ops.packed_columns(d)
    for i in range(4):
        m = new[i]
        rows, slots = slice(at, at + m), torch.arange(before[i], before[i] + m, device="cuda")
        y, _ = _rotate(k[rows].double(), cos[seen[i]: seen[i] + m], sin[seen[i]: seen[i] + m], 0)
        for pages, old, x, unit, out in ((kp, k0, y, units[0], k_out), (vp, v0, v[rows].double(), units[1], v_out)):
            code, scale, value = _quantise(x, unit)
            code_, scale_, value_ = _stored(pages, table[i], d, size, slots)
            assert torch.equal(scale_[..., : scale.shape[-1]], scale) and not bool(scale_[..., scale.shape[-1]:].any())
            assert torch.equal(code_[..., :d], code) and not bool(code_[..., d:].any())
            # back out of the pages: the values, rounded once more where the unit has more bits
            back = (value_.float() * torch.tensor(unit, device="cuda")).to(dt)
            assert bool(torch.isnan(out[rows]).eq(torch.isnan(back)).all()) and torch.equal(out[rows].nan_to_num(7.0), back.nan_to_num(7.0))
            # nothing else was written
            where = (table[i].long()[slots // size], slice(None), slots % size // 16)
            for part, w in ((slice(0, 8 * p), p // 2), (slice(8 * p, 9 * p), p // 16)):
                a, b = (z.view(n, g, size // 16, 9 * p)[..., part].unflatten(-1, (16, w)) for z in (pages, old))
                b[where + (slots % 16,)] = a[where + (slots % 16,)]
        at += m
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("g, d, size", [(2, 128, 16), (3, 40, 32), (1, 37, 16)])
def test_gather_of_ranges(dt, four, g, d, size):
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    lens = [70, 0, 33, 100]
    table, n = _page_table(4, 7, 3, 1)
    zero = _i32(0, 0, 0, 0)
    rows = _rnd(2, sum(lens), g, d, dt=dt)
    if four:
        kp, vp = (torch.zeros(n, g, ops.packed_page_bytes(size, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        kp, vp = (torch.zeros(n, size, g, d, dtype=dt, device="cuda") for _ in range(2))
    cu = torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    ops.paged_append_rope(rows, -rows, kp, vp, table, zero, cu_seqlens=cu)
    value = _quantise(rows.double())[2].to(dt) if four else rows
    for first, take in ((None, [5, 0, 33, 1]), ([0, 0, 10, 37], [70, 0, 20, 62])):
        cq = torch.tensor([0] + take, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        k, v = (torch.full((sum(take) + 2, g + 1, d), 4.0, dtype=dt, device="cuda")[:, 1:] for _ in range(2))
        ops.paged_gather(kp, vp, table, _i32(*lens), cq, k, v, first=None if first is None else _i32(*first))
        ops.check_status(k.device)
        at = 0
        for i, m in enumerate(take):
            lo = int(cu[i]) + (lens[i] - m if first is None else first[i])
            assert torch.equal(k[at: at + m], value[lo: lo + m]) and torch.equal(v[at: at + m], -value[lo: lo + m])
            at += m
        assert bool((k[at:] == 4).all()) and bool((v[at:] == 4).all())
    # slots that are none
    k, v = (torch.full((4, g, d), 4.0, dtype=dt, device="cuda") for _ in range(2))
    ops.paged_gather(kp, vp, table, _i32(*lens), _i32(0, 2, 3, 4, 4), k, v, first=_i32(69, 0, -1, 0))
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(k.device)
    assert torch.equal(k[0], value[69]) and not bool(k[1:].any()) and not bool(v[1:].any())


# ---------------------------------------------------------------------------------------
# one-token attention over 4-bit pages
# ---------------------------------------------------------------------------------------

LENS = [0, 1, 15, 16, 17, 63, 64, 65, 333, 1100]


def _cache4(lens, g, d, size, seed, units=(1.0, 1.0), layout="plain"):
    """4-bit pages with rows of standard normal keys and values; all else is codes and scales of NaN.  Also the values."""
    from project_chronos_b200 import ops
    nbytes = ops.packed_page_bytes(size, d)
    width = max(1, -(-max(lens) // size)) + 1
    table, n = _page_table(len(lens), width, 2, seed)
    if layout == "plain":
        kp, vp = (torch.full((n, g, nbytes), 0x7F, dtype=torch.uint8, device="cuda") for _ in range(2))
    else:   # keys and values of a page side by side, heads apart
        both = torch.full((g, n, 2, nbytes + 16), 0x7F, dtype=torch.uint8, device="cuda")
        kp, vp = (both[:, :, i, 16:].transpose(0, 1) for i in range(2))
    x = _rnd(seed + 1, sum(lens), 2, g, d)
    cu = torch.tensor([0] + list(lens), dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    ops.paged_append_rope(x[:, 0], x[:, 1], kp, vp, table, torch.zeros_like(cu[1:]), cu_seqlens=cu, k_scale=units[0], v_scale=units[1])
    ops.check_status(x.device)
    rows = []
    for i, m in enumerate(lens):
        slots = torch.arange(m, device="cuda")
        k, v = (_stored(p.contiguous(), table[i], d, size, slots)[2] * float(torch.tensor(u)) for p, u in ((kp, units[0]), (vp, units[1])))
        rows.append((k, v))
    return kp, vp, table, _i32(*lens), rows


def _visible(n, window, sinks):
    j = torch.arange(n, device="cuda")
    return (j >= n - window) | (j < sinks) if window else j >= 0


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d, size", [(8, 2, 128, 16), (4, 4, 64, 64), (10, 2, 80, 48), (9, 1, 96, 16), (17, 1, 128, 32), (16, 2, 256, 16),
                                           (24, 2, 256, 32), (20, 2, 64, 16), (6, 3, 40, 16), (2, 1, 37, 48), (3, 3, 1, 16), (40, 1, 8, 16)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 0), (64, 4), (7, 100)])
def test_decode4_matches_its_definition(dt, h, g, d, size, window, sinks):
    from project_chronos_b200 import ops
    units = (1.0, 1.0) if h % 2 else (0.5, 3.1)
    kp, vp, table, lens, rows = _cache4(LENS, g, d, size, h * d + size, units, "plain" if h % 4 else "side by side")
    q = _rnd(3, len(LENS), h, d, dt=dt, scale=2.0 / units[0])
    lse = torch.full((len(LENS), h), 7.0, device="cuda")
    out = ops.paged_attn_decode4(q, kp, vp, table, lens, window=window, sinks=sinks, k_scale=units[0], v_scale=units[1], lse=lse)
    ops.check_status(out.device)
    for b, (k, v) in enumerate(rows):
        seen = _visible(LENS[b], window, sinks)
        _check_attention(out[b], lse[b], q[b], k[seen], v[seen], d ** -0.5, dt, True)
        if LENS[b] == 0:
            assert not bool(out[b].any())


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h, g, lens", [(8, 1, [20011]), (4, 2, [1, 9000, 3, 0, 5000]), (24, 1, [7001, 64]), (32, 8, [3000] * 40)])
def test_decode4_split_over_the_length(dt, h, g, lens):
    from project_chronos_b200 import ops
    d = 128
    kp, vp, table, ln, rows = _cache4(lens, g, d, 16, 5)
    q = _rnd(6, len(lens), h, d, dt=dt, scale=3.0)
    lse = torch.empty(len(lens), h, device="cuda")
    out = ops.paged_attn_decode4(q, kp, vp, table, ln, lse=lse)
    assert torch.equal(out, ops.paged_attn_decode4(q, kp, vp, table, ln))
    for b, (k, v) in enumerate(rows):
        _check_attention(out[b], lse[b], q[b], k, v, d ** -0.5, dt, True)
    over = q.clone()
    assert ops.paged_attn_decode4(over, kp, vp, table, ln, out=over) is over and torch.equal(over, out)


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_decode4_of_queries_of_all_sizes(dt):
    """Heads of large, tiny and mixed columns, of zeros, and one that is not finite."""
    from project_chronos_b200 import ops
    h, g, d = 8, 2, 128
    kp, vp, table, ln, rows = _cache4([200, 77], g, d, 16, 5)
    q = _rnd(6, 2, h, d)
    q[:, 0] *= 1e-3
    q[:, 1] *= 200.0
    q[:, 2] = 0.0
    q[:, 3, 1:] *= 1e-4
    q[:, 4] *= 0.0 if dt == HF else 1e-30
    q = q.to(dt)
    lse = torch.empty(2, h, device="cuda")
    out = ops.paged_attn_decode4(q, kp, vp, table, ln, lse=lse)
    for b, (k, v) in enumerate(rows):
        _check_attention(out[b], lse[b], q[b], k, v, d ** -0.5, dt, True)
    bad = q.clone()
    bad[0, 5, 9] = math.nan
    got = ops.paged_attn_decode4(bad, kp, vp, table, ln)
    assert bool(torch.isnan(got[0, 5]).all())
    keep = [i for i in range(h) if i != 5]
    assert torch.equal(got[0, keep], out[0, keep]) and torch.equal(got[1], out[1])


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_decode4_of_odd_strides_and_bad_pages(dt):
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    h, g, d, lens = 6, 2, 64, [100, 40]
    kp, vp, table, ln, rows = _cache4(lens, g, d, 16, 9)
    q = _rnd(3, 2, h + 1, d + 3, dt=dt)[:, 1:, 3:]
    out = torch.full((2, h, 2 * d + 1), 3.0, dtype=dt, device="cuda")
    ops.paged_attn_decode4(q, kp, vp, table, ln, out=out[..., 1: d + 1])
    for b, (k, v) in enumerate(rows):
        _check_attention(out[b, :, 1: d + 1], None, q[b], k, v, d ** -0.5, dt, True)
    assert bool((out[..., 0] == 3).all()) and bool((out[..., d + 1:] == 3).all())
    broken = table.clone()
    broken[0, 2] = -1
    broken[1, 1] = kp.shape[0]
    got = ops.paged_attn_decode4(q, kp, vp, broken, ln)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(out.device)
    for b, (k, v) in enumerate(rows):
        seen = torch.arange(lens[b], device="cuda") // 16 != 2 - b
        _check_attention(got[b], None, q[b], k[seen], v[seen], d ** -0.5, dt, True)
    got = ops.paged_attn_decode4(q, kp, vp, table, _i32(-3, 10 ** 6))     # behind the table: cut to it
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(out.device)
    assert not bool(got[0].any())


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_decode4_far_below_the_heaviest(dt):
    """Very many slots 2^-20 as heavy as the first still count."""
    from project_chronos_b200 import ops
    n, d, size = 40000, 64, 16
    x = torch.zeros(n, 2, 1, d, device="cuda")
    x[0, 0, 0, :16] = 6.0                              # scores 6 * 16 * q against 0
    x[:, 1, 0, 0] = 6.0
    x[0, 1] = 0.0
    table = torch.arange(n // size, dtype=torch.int32, device="cuda").view(1, -1)
    kp, vp = (torch.zeros(n // size, 1, ops.packed_page_bytes(size, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    ops.paged_append_rope(x[:, 0], x[:, 1], kp, vp, table, _i32(0), cu_seqlens=_i32(0, n))
    q = torch.zeros(1, 1, d, dtype=dt, device="cuda")
    q[..., :16] = 20 * math.log(2) / 96                # about 2^-20 each: together 3.7 %
    out = ops.paged_attn_decode4(q, kp, vp, table, _i32(n), scale=1.0)
    _check_attention(out[0], None, q[0], x[:, 0], x[:, 1], 1.0, dt, True)


# ---------------------------------------------------------------------------------------
# page bounds
# ---------------------------------------------------------------------------------------

def _bounds_of(k, size):
    """Keys [n, G, D] of one sequence: [pages, 2, G, D]."""
    return torch.stack([torch.stack([c.amin(0), c.amax(0)]) for c in k.split(size)])


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("g, d, size", [(2, 128, 16), (3, 64, 64), (1, 80, 48), (1, 256, 128), (2, 37, 16)])
@pytest.mark.parametrize("step", [1, 23])
def test_bounds_follow_the_appends(dt, four, g, d, size, step):
    """Token by token and in packed chunks, against the smallest and largest of the slots; then from nothing."""
    from project_chronos_b200 import PagedCache, ops
    c = PagedCache(3, 30, g, d, 9, "cuda", dt, page_size=size, four_bit=four, page_bounds=True, k_scale=0.5)
    c.bounds.fill_(math.nan)                           # what earlier owners left
    for b in range(3):
        c.reserve(b, 140)
    book = [[], [], []]
    for i in range(140 // max(step, 2)):
        new = [1, 1, 1] if step == 1 else [step, i % 2 * 7, 1]
        t = sum(new)
        k, v = _rnd(100 + i, t, g, d, dt=dt), _rnd(i, t, g, d, dt=dt)
        cu = None if step == 1 else torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        c.append(k, v, cu)
        for b, part in enumerate(k.split(new)):
            book[b].append(part)
    ops.check_status(c.lens.device)
    def check():
        for b in range(3):
            rows = torch.cat(book[b])
            if four:
                rows = _quantise(rows.double(), 0.5)[2].to(dt)
            want = _bounds_of(rows, size)
            got = c.bounds[c.page_table[b, : want.shape[0]].long()]
            assert torch.equal(got, want)
    check()
    c.bounds.fill_(math.nan)
    ops.paged_bounds(c.k_pages, c.bounds, c.page_table, c.lens, full=True, k_scale=c.k_scale)
    check()


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_bounds_of_keys_that_are_not_finite(dt):
    from project_chronos_b200 import ops
    size, g, d = 16, 2, 64
    kp = _rnd(1, 4, size, g, d, dt=dt)
    kp[2, 3, 0, 5], kp[2, 4, 1, 6], kp[2, 5, 1, 7] = math.nan, math.inf, -math.inf
    bounds = torch.zeros(4, 2, g, d, dtype=dt, device="cuda")
    ops.paged_bounds(kp, bounds, _i32(2).view(1, 1), _i32(12), full=True)
    want = torch.stack([kp[2, :12].amin(0), kp[2, :12].amax(0)])
    assert torch.equal(torch.isnan(bounds[2]), torch.isnan(want)) and bool(torch.isnan(bounds[2, :, 0, 5]).all())
    assert torch.equal(bounds[2].nan_to_num(9.0, 8.0, -8.0), want.nan_to_num(9.0, 8.0, -8.0))
    assert not bool(bounds[[0, 1, 3]].any())
    from project_chronos_b200 import _native as N
    ops.paged_bounds(kp, bounds, _i32(2, 77).view(1, 2), _i32(40), cu_seqlens=_i32(0, 30))
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(kp.device)


# ---------------------------------------------------------------------------------------
# selected pages
# ---------------------------------------------------------------------------------------

def _selected(q, lo, hi, g, topk, first, last):
    """The pages of one token: q [H, D], lo and hi [m, G, D] -> [G, topk]."""
    m, h = lo.shape[0], q.shape[0]
    res = torch.full((g, topk), -1, dtype=torch.int32)
    for i in range(g):
        x = q[i * h // g: (i + 1) * h // g].double()
        up, down = x.clamp(min=0).nan_to_num(math.nan).sum(0), x.clamp(max=0).sum(0)
        score = (up * hi[:, i].double() + down * lo[:, i].double()).sum(1).cpu().tolist() if m else []
        def rank(j):
            if j < first or j >= m - last:
                return (0, 0.0, j)
            return (1, 0.0, j) if math.isnan(score[j]) else (2, -score[j], j)
        best = sorted(sorted(range(m), key=rank)[:topk])
        res[i, : len(best)] = torch.tensor(best, dtype=torch.int32)
    return res


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d", [(8, 2, 128), (4, 4, 64), (9, 1, 96), (16, 2, 256), (6, 3, 37), (2, 1, 1)])
@pytest.mark.parametrize("topk, first, last", [(1, 0, 1), (8, 1, 2), (40, 3, 37), (16, 0, 1)])
@pytest.mark.parametrize("new", [None, [1, 9, 0, 17, 3]])
def test_select_matches_its_definition(dt, h, g, d, topk, first, last, new):
    from project_chronos_b200 import ops
    size = 4
    lens = [0 if new is None else 1, 61, 160, 999, 3000]
    b = len(lens)
    table, n = _page_table(b, 760, 1, 1)
    bounds = _rnd(2, n, 2, g, d, dt=dt).sort(dim=1).values.contiguous()
    t = b if new is None else sum(new)
    pad = 0 if new is None else 2
    q = _rnd(3, t + pad, h, d + 1, dt=dt)[..., 1:]
    cu = None if new is None else torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    out = torch.full((t + pad, g, topk), -7, dtype=torch.int32, device="cuda")
    assert ops.paged_select(q, bounds, table, _i32(*lens), size, topk, first=first, last=last, cu_seqlens=cu, out=out) is out
    ops.check_status(out.device)
    row = 0
    for i in range(b):
        for j in range(1 if new is None else new[i]):
            at = lens[i] if new is None else lens[i] - new[i] + 1 + j
            m = -(-max(at, 0) // size)
            x = bounds[table[i, :m].long()]
            assert torch.equal(out[row].cpu(), _selected(q[row], x[:, 0], x[:, 1], g, topk, first, last)), (i, j)
            row += 1
    assert bool((out[row:] == -7).all())


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_select_orders_ties_and_what_is_not_a_number(dt):
    """Equal scores go by the lower page; NaN comes first, pages that are none last."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    h, g, d, m = 4, 2, 64, 500
    table = torch.arange(m, dtype=torch.int32, device="cuda").view(1, m)
    ln = _i32(m * 16)
    pick = lambda q, bounds, k, tab=table: ops.paged_select(q, bounds, tab, ln, 16, k, first=1, last=1)[0].tolist()  # noqa: E731
    few = _rnd(1, 3, 2, g, d, dt=dt).sort(dim=1).values
    bounds = few[torch.randint(0, 3, (m,), generator=_gen(2), device="cuda")].contiguous()      # three kinds of page
    q = _rnd(3, 1, h, d, dt=dt)
    for k in (2, 3, 100, 200, 400, 499):
        want = _selected(q[0], bounds[:, 0], bounds[:, 1], g, k, 1, 1).tolist()
        assert pick(q, bounds, k) == want
    for zero in (torch.zeros_like(q), -torch.zeros_like(q)):                                    # all equal
        assert pick(zero, bounds, 7) == [[0, 1, 2, 3, 4, 5, 499]] * g
    odd = bounds.clone()
    odd[77, 1, 0, 3], odd[300, 0, 1, 3] = math.nan, math.nan
    got = pick(q, odd, 3)
    assert got == [[0, 77, 499], [0, 300, 499]]
    odd = bounds.clone()
    odd[:, :, :, 0] = torch.tensor([-math.inf, math.inf], device="cuda")[None, :, None].to(dt)  # infinite: all equal
    assert pick(q.abs() + 0.1, odd, 4) == [[0, 1, 2, 499]] * g
    broken = table.clone()
    broken[0, ::2] = -1
    got = pick(q, bounds, 200, broken)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(q.device)
    assert all(x % 2 == 1 or x in (0, 499) for row in got for x in row)


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("scale", [1.0, 1e-6])
def test_select_of_very_many_pages(dt, scale):
    """More pages than shared memory holds the keys of, more tokens than the workspace holds at once; scores that
    32 bits would mix up."""
    from project_chronos_b200 import ops
    h, g, d, m = 2, 1, 16, 20000
    bounds = (1.0 + scale * _rnd(1, m, 2, g, d)).to(dt).contiguous()
    table = torch.randperm(m, generator=_gen(2), device="cuda").to(torch.int32).view(1, m)
    t = 1700                                              # 272 MB of keys
    q = _rnd(3, t, h, d, dt=dt).abs()
    ln = _i32(m)
    out = ops.paged_select(q, bounds, table, ln, 1, 33, first=2, last=3, cu_seqlens=_i32(0, t))
    for row in (0, 1, 850, t - 1):
        n = m - (t - 1 - row)
        x = bounds[table[0, :n].long()]
        assert torch.equal(out[row].cpu(), _selected(q[row], x[:, 0], x[:, 1], g, 33, 2, 3)), row


# ---------------------------------------------------------------------------------------
# attention over selected pages
# ---------------------------------------------------------------------------------------

def _cache16(lens, g, d, size, dt, seed, layout="plain"):
    width = max(1, -(-max(lens) // size)) + 1
    table, n = _page_table(len(lens), width, 2, seed)
    shape = (n, size, g, d + (1 if layout == "odd" else 0))
    kp, vp = (torch.full(shape, math.nan, dtype=dt, device="cuda")[..., :d] for _ in range(2))
    rows = []
    for i, m in enumerate(lens):
        k, v = _rnd(seed + 2 * i, m, g, d, dt=dt), _rnd(seed + 2 * i + 1, m, g, d, dt=dt)
        s = torch.arange(m, device="cuda")
        kp[table[i].long()[s // size], s % size], vp[table[i].long()[s // size], s % size] = k, v
        rows.append((k.double(), v.double()))
    return kp, vp, table, _i32(*lens), rows


def _slots(ids, size, n):
    """Slots below n of the listed pages, one after the other."""
    m = -(-n // size)
    parts = [torch.arange(i * size, min(n, (i + 1) * size), device="cuda") for i in ids if 0 <= i < m]
    return torch.cat(parts) if parts else torch.empty(0, dtype=torch.long, device="cuda")


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d, size, kind", [
    (8, 2, 128, 16, "plain"), (4, 4, 64, 64, "plain"), (10, 2, 80, 48, "plain"), (17, 1, 128, 32, "plain"), (16, 2, 256, 16, "plain"),
    (6, 3, 40, 7, "plain"), (8, 2, 128, 20, "plain"), (2, 1, 37, 5, "plain"), (40, 1, 8, 16, "plain"), (8, 2, 64, 16, "odd"), (3, 3, 1, 1, "plain"),
    (8, 2, 128, 16, "four"), (4, 4, 64, 64, "four"), (10, 2, 80, 48, "four"), (17, 1, 128, 32, "four"), (24, 2, 256, 16, "four"), (2, 1, 37, 16, "four")])
@pytest.mark.parametrize("new", [None, [1, 4, 0, 9]])
def test_sparse_attention_matches_its_definition(dt, h, g, d, size, kind, new):
    """Lists in any order, with entries that are none, pages behind the token, one named twice."""
    from project_chronos_b200 import ops
    lens = [1, 50, 333, 1100]
    kp, vp, table, ln, rows = _cache4(lens, g, d, size, 7) if kind == "four" else _cache16(lens, g, d, size, dt, 7, kind)
    b, topk = len(lens), 9
    t = b if new is None else sum(new)
    pad = 0 if new is None else 2
    cu = None if new is None else torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    q = _rnd(5, t + pad, h, d, dt=dt, scale=2.0)
    most = max(-(-n // size) for n in lens)
    pages = torch.randint(-2, most + 3, (t + pad, g, topk), generator=_gen(6), device="cuda").to(torch.int32)
    pages[:, 0, :3] = _i32(0, 0, -1)
    pages[0, g - 1] = -1                                  # nothing at all
    out = torch.full((t + pad, h, d), 3.0, dtype=dt, device="cuda")
    lse = torch.full((t + pad, h), 3.0, device="cuda")
    ops.paged_attn_sparse(q, kp, vp, table, ln, pages, cu_seqlens=cu, out=out, lse=lse)
    ops.check_status(out.device)
    row = 0
    for i in range(b):
        k, v = rows[i]
        for j in range(1 if new is None else new[i]):
            n = lens[i] if new is None else lens[i] - new[i] + 1 + j
            for x in range(g):
                s = _slots(pages[row, x].tolist(), size, n)
                heads = slice(x * h // g, (x + 1) * h // g)
                _check_attention(out[row, heads], lse[row, heads], q[row, heads], k[s][:, x: x + 1], v[s][:, x: x + 1], d ** -0.5, dt, kind == "four")
                if s.numel() == 0:
                    assert not bool(out[row, heads].any())
            row += 1
    assert bool((out[row:] == 3).all()) and bool((lse[row:] == 3).all())
    over = q.clone()
    ops.paged_attn_sparse(over, kp, vp, table, ln, pages, cu_seqlens=cu, out=over)
    assert torch.equal(over[:row], out[:row])


@gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("tokens", [1, 3, 600])
def test_sparse_attention_over_all_pages_is_attention(four, tokens):
    """Few tokens (a cluster each) and many (a block each)."""
    from project_chronos_b200 import ops
    h, g, d, size, dt, n = 8, 2, 128, 16, BF, 2000
    kp, vp, table, ln, rows = _cache4([n], g, d, size, 3) if four else _cache16([n], g, d, size, dt, 3)
    q = _rnd(4, tokens, h, d, dt=dt, scale=2.0)
    pages = torch.arange(125, dtype=torch.int32, device="cuda").expand(tokens, g, 125).contiguous()
    out = ops.paged_attn_sparse(q, kp, vp, table, ln, pages, cu_seqlens=_i32(0, tokens))
    k, v = rows[0]
    for t in {0, tokens // 2, tokens - 1}:
        m = n - (tokens - 1 - t)
        _check_attention(out[t], None, q[t], k[:m], v[:m], d ** -0.5, dt, four)


@gpu
@pytest.mark.parametrize("four", [False, True])
def test_sparse_attention_of_bad_pages_and_lengths(four):
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    h, g, d, size, dt = 8, 2, 64, 16, BF
    kp, vp, table, ln, rows = _cache4([100, 90], g, d, size, 3) if four else _cache16([100, 90], g, d, size, dt, 3)
    q = _rnd(4, 2, h, d, dt=dt)
    pages = torch.arange(3, dtype=torch.int32, device="cuda").expand(2, g, 3).contiguous()
    table = table.clone()
    table[0, 1], table[1, 0] = -5, kp.shape[0] + 1
    out = ops.paged_attn_sparse(q, kp, vp, table, ln, pages)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(q.device)
    for b, gone in ((0, 1), (1, 0)):
        seen = torch.arange(48, device="cuda") // 16 != gone
        _check_attention(out[b], None, q[b], rows[b][0][:48][seen], rows[b][1][:48][seen], d ** -0.5, dt, four)
    out = ops.paged_attn_sparse(q, kp, vp, table, _i32(-1, 0), pages)
    with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
        ops.check_status(q.device)
    assert not bool(out.any())
    none = ops.paged_attn_sparse(q, kp, vp, table, ln, pages[:, :, :0].contiguous())
    ops.check_status(q.device)
    assert not bool(none.any())


# ---------------------------------------------------------------------------------------
# refusals of the torch-facing calls
# ---------------------------------------------------------------------------------------

@gpu
def test_calls_refuse_what_they_cannot_take():
    from project_chronos_b200 import ops
    kp, vp, table, ln, _ = _cache16([20, 30], 2, 64, 16, BF, 1)
    k4, v4, t4, l4, _ = _cache4([20, 30], 2, 64, 16, 1)
    k, q = _rnd(1, 2, 2, 64, dt=BF), _rnd(2, 2, 4, 64, dt=BF)
    cos, sin = _tables(64, 64)
    bounds = torch.zeros(kp.shape[0], 2, 2, 64, dtype=BF, device="cuda")
    pages = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    rope = lambda **kw: ops.paged_append_rope(**{**dict(k=k, v=k, k_pages=kp, v_pages=vp, page_table=table, lens=ln, seen=ln, cos=cos, sin=sin), **kw})  # noqa: E731
    for kw, err, text in ((dict(k=k.float(), v=k.float()), TypeError, "expected"), (dict(v=k[:1]), ValueError, "must be"),
                          (dict(cos=None), ValueError, "together"), (dict(seen=None), ValueError, "seen"), (dict(q_out=q), ValueError, "needs q"),
                          (dict(cos=cos.half(), sin=sin.half()), TypeError, "fp32"), (dict(sin=sin[:5]), ValueError, "must be"),
                          (dict(k_pages=k4, v_pages=kp), (TypeError, ValueError), "must be|expected|multiple"), (dict(k_pages=kp.expand(kp.shape).as_strided(kp.shape, (0, 128, 64, 1))), ValueError, "expanded"),
                          (dict(k=k.clone().requires_grad_()), RuntimeError, "forward-only"), (dict(lens=ln.long()), TypeError, "int32"),
                          (dict(k_pages=k4[..., :100].contiguous(), v_pages=v4[..., :100].contiguous()), ValueError, "multiple of"),
                          (dict(rope_start=8), Exception, "rotation"), (dict(k_pages=k4, v_pages=v4, page_table=t4, k_scale=0.0), Exception, "k_scale")):
        with pytest.raises(err, match=text):
            rope(**kw)
    with pytest.raises(TypeError, match="uint8"):
        ops.paged_attn_decode4(q, kp, vp, table, ln)
    with pytest.raises(ValueError, match="must be"):
        ops.paged_attn_decode4(q[:1], k4, v4, t4, l4)
    with pytest.raises(Exception, match="heads"):
        ops.paged_attn_decode4(q[:, :3], k4, v4, t4, l4)
    with pytest.raises(ValueError, match="32 bits"):
        ops.paged_attn_decode4(q, k4, v4, t4, l4, window=1 << 31)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_gather(kp, vp, table, ln, _i32(0, 1, 2), kp[0, :2], k.clone())
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_gather(kp, vp, table, ln, _i32(0, 1, 2), k, k)
    with pytest.raises(ValueError, match="expanded"):
        ops.paged_gather(kp, vp, table, ln, _i32(0, 1, 2), k[:1].expand(2, 2, 64), k.clone())
    with pytest.raises(ValueError, match="must be"):
        ops.paged_bounds(kp, bounds[1:], table, ln)
    with pytest.raises(TypeError, match="expected"):
        ops.paged_bounds(kp, bounds.float(), table, ln)
    for kw, err, text in ((dict(topk=0), ValueError, "topk"), (dict(topk=2, first=1, last=2), Exception, "topk"), (dict(last=0), Exception, "topk"),
                          (dict(bounds=bounds.float()), TypeError, "expected"), (dict(q=q[:1]), Exception, "rows"),
                          (dict(out=pages.long()), TypeError, "int32"), (dict(topk=1 << 40), ValueError, "32 bits"), (dict(page_size=0), Exception, "page_size")):
        with pytest.raises(err, match=text):
            ops.paged_select(**{**dict(q=q, bounds=bounds, page_table=table, lens=ln, page_size=16, topk=3), **kw})
    for kw, err, text in ((dict(pages=pages.long()), TypeError, "int32"), (dict(pages=pages[:1]), ValueError, "must be"),
                          (dict(q=q.float()), TypeError, "expected"), (dict(out=q[:, :1].expand(q.shape)), ValueError, "expanded"),
                          (dict(scale=0.0), Exception, "scale")):
        with pytest.raises(err, match=text):
            ops.paged_attn_sparse(**{**dict(q=q, k_pages=kp, v_pages=vp, page_table=table, lens=ln, pages=pages), **kw})


# ---------------------------------------------------------------------------------------
# together, as they are used
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("dt", [BF, FP])
def test_prompts_chunks_and_steps_of_a_cache(four, dt):
    """Prompts rotated into the cache, a second chunk that attends to the cached rows, then single tokens with
    attention over all slots and over selected pages."""
    from project_chronos_b200 import PagedCache, ops
    h, g, d, size = 8, 2, 64, 16
    c = PagedCache(3, 60, g, d, 20, "cuda", dt, page_size=size, four_bit=four, page_bounds=True)
    cos, sin = _tables(320, d)
    for b in range(3):
        c.reserve(b, 300)
    book_k, book_v = [[], [], []], [[], [], []]
    def keep(k, v, new, start):
        for b, (x, y) in enumerate(zip(k.split(new), v.split(new))):
            x = _rotate(x.double(), cos[start[b]: start[b] + new[b]], sin[start[b]: start[b] + new[b]], 0)[0]
            book_k[b].append(_quantise(x)[2] if four else x.to(dt).double())
            book_v[b].append(_quantise(y.double())[2] if four else y.double())
    start = [0, 0, 0]
    for chunk, new in enumerate(([100, 1, 40], [60, 90, 0])):
        t = sum(new)
        q, k, v = (_rnd(10 * chunk + i, t, x, d, dt=dt) for i, x in ((1, h), (2, g), (3, g)))
        cu = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        q = c.append_rope(q, k, v, cos, sin, cu_seqlens=cu)
        keep(k, v, new, start)
        start = [a + n for a, n in zip(start, new)]
        ck = torch.tensor([0] + start, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        ka, va = c.gather(ck, sum(start) + 1)
        for b in range(3):
            lo = int(ck[b])
            if not four and dt != FP:                     # equal but for the rotation's rounding
                assert float((ka[lo: lo + start[b]].double() - torch.cat(book_k[b])).abs().max()) <= 2.0 ** -5
            else:
                assert torch.allclose(ka[lo: lo + start[b]].double(), torch.cat(book_k[b]), rtol=2.0 ** -8 if dt == BF else 2.0 ** -20, atol=2.0 ** -20)
            assert torch.equal(va[lo: lo + start[b]].double(), torch.cat(book_v[b]).to(dt).double())
        assert not bool(ka[sum(start):].any())
        out = ops.window_attention(q, ka, va, cu, cu_seqlens_k=ck)
        ops.check_status(out.device)
        at = 0
        for b, n in enumerate(new):
            for j in {0, n - 1} if n else ():
                m = start[b] - n + j + 1
                lo = int(ck[b])
                _check_attention(out[at + j], None, q[at + j], ka[lo: lo + m], va[lo: lo + m], d ** -0.5, dt, False)
            at += n
    for step in range(20):
        q, k, v = (_rnd(100 + 10 * step + i, 3, x, d, dt=dt) for i, x in ((1, h), (2, g), (3, g)))
        q = c.append_rope(q, k, v, cos, sin)
        keep(k, v, [1, 1, 1], start)
        start = [a + 1 for a in start]
        out = c.attend(q)
        some, pages = c.attend_sparse(q, 6, first=1, last=2)
        every, _ = c.attend_sparse(q, 20)
        ops.check_status(out.device)
        ck = torch.tensor([0] + start, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        ka, va = c.gather(ck, sum(start))
        for b in range(3):
            lo, n = int(ck[b]), start[b]
            kb, vb = ka[lo: lo + n], va[lo: lo + n]
            _check_attention(out[b], None, q[b], kb, vb, d ** -0.5, dt, four)
            _check_attention(every[b], None, q[b], kb, vb, d ** -0.5, dt, four)
            want = _bounds_of(kb, size)
            assert torch.equal(c.bounds[c.page_table[b, : want.shape[0]].long()], want)
            assert torch.equal(pages[b].cpu(), _selected(q[b], want[:, 0], want[:, 1], g, 6, 1, 2))
            for x in range(g):
                s = _slots(pages[b, x].tolist(), size, n)
                heads = slice(x * h // g, (x + 1) * h // g)
                _check_attention(some[b, heads], None, q[b, heads], kb[s][:, x: x + 1], vb[s][:, x: x + 1], d ** -0.5, dt, four)
    assert c.lens.tolist() == start == c.seen.tolist()


@gpu
@pytest.mark.parametrize("four", [False, True])
def test_a_captured_step_of_rotation_and_selection(four):
    """One graph for a step, replayed while rows grow, one that fills up and one that is released and starts again;
    a second graph with workspaces of its own replayed in between."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import PagedCache, ops
    h, g, d, dt, size = 8, 2, 64, BF, 16
    make = lambda: PagedCache(2, 24, g, d, 12, "cuda", dt, page_size=size, four_bit=four, page_bounds=True)  # noqa: E731
    cos, sin = _tables(400, d)
    live, ref = make(), make()
    other = make()
    rows = {c: [torch.zeros(2, x, d, dtype=dt, device="cuda") for x in (h, g, g)] for c in (live, other)}
    outs = {}

    def step(c, q, k, v):
        q = c.append_rope(q, k, v, cos, sin)
        return c.attend(q), *c.attend_sparse(q, 3, first=1, last=1)

    graphs = {}
    for c in (live, other):
        for b in range(2):
            c.reserve(b, 32 + 100 * b)
        step(c, *rows[c])                                 # outside the capture first
        for b in range(2):
            c.release(b)
            c.reserve(b, 32 + 100 * b)
        torch.cuda.synchronize()
        graphs[c] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[c]):
            outs[c] = step(c, *rows[c])
        assert c.lens.tolist() == [0, 0]
    ops.check_status(live.lens.device)
    for b in range(2):
        ref.reserve(b, 32 + 100 * b)
    gen = _gen(5)
    for i in range(80):
        if i == 36:
            for c in (live, ref):
                c.reserve(0, 50)
        if i == 60:
            for c in (live, ref):
                c.release(1)
                c.reserve(1, 40)
        for x in rows[live]:
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        graphs[live].replay()
        if i < 30:
            graphs[other].replay()
        want = step(ref, *(x.clone() for x in rows[live]))
        full = 32 <= i < 36 or i >= 68                    # row 0 of 32, then of 64 slots
        for a, b in zip(outs[live], want):
            assert torch.equal(a, b)
        assert live.lens.tolist() == ref.lens.tolist() and torch.equal(live.bounds, ref.bounds)
        if full:
            with pytest.raises(N.ChronosMoeError, match="INVALID_ARG"):
                ops.check_status(live.lens.device)
        else:
            ops.check_status(live.lens.device)


@gpu
def test_calls_follow_the_current_stream():
    """On another stream, behind work that is still running there."""
    from project_chronos_b200 import PagedCache, ops
    h, g, d, dt = 8, 2, 128, BF
    cos, sin = _tables(4200, d)
    q, k, v = (_rnd(i, 4096, x, d, dt=dt) for i, x in ((1, h), (2, g), (3, g)))
    cu = _i32(0, 4096)
    res = []
    for stream in (None, torch.cuda.Stream()):
        c = PagedCache(1, 70, g, d, 70, "cuda", dt, page_size=64, four_bit=True, page_bounds=True)
        c.reserve(0, 4200)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(10):
                big = big @ big * 0.01
            late = [x * 1.0 for x in (q, k, v)]
            qr = c.append_rope(*late, cos, sin, cu_seqlens=cu)
            out, pages = c.attend_sparse(qr[-3:].contiguous(), 9, cu_seqlens=_i32(0, 3))
            one = c.attend(qr[-1:])
        torch.cuda.synchronize()
        res.append((qr, out, pages, one))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    ops.check_status(q.device)


# ---------------------------------------------------------------------------------------
# many rows, views, streams, other parts of the cache
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("four", [False, True])
def test_very_many_rows(dt, four):
    """More rows than a grid's second dimension takes, and than run at once."""
    from project_chronos_b200 import ops
    b, h, g, d, size = 70000, 2, 1, 16, 16
    k, v = _rnd(1, b, g, d, dt=dt), _rnd(2, b, g, d, dt=dt)
    q = _rnd(3, b, h, d, dt=dt)
    if four:
        kp, vp = (torch.zeros(2 * b, g, ops.packed_page_bytes(size, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        kp, vp = (torch.zeros(2 * b, size, g, d, dtype=dt, device="cuda") for _ in range(2))
    table = torch.randperm(2 * b, generator=_gen(4), device="cuda").to(torch.int32).view(b, 2)
    ln = torch.full((b,), 15, dtype=torch.int32, device="cuda")
    ln[1::2] = 16                                          # the second page's first slot
    ops.paged_append_rope(k, v, kp, vp, table, ln, lens_out=ln)
    bounds = torch.zeros(2 * b, 2, g, d, dtype=dt, device="cuda")
    ops.paged_bounds(kp, bounds, table, ln, full=True)
    pages = ops.paged_select(q, bounds, table, ln, size, 1)
    want = torch.zeros(b, 1, 1, dtype=torch.int32, device="cuda")
    want[1::2] = 1                                         # a token's own page
    assert torch.equal(pages, want)
    out = ops.paged_attn_sparse(q, kp, vp, table, ln, pages)
    ops.check_status(out.device)
    values = _quantise(v.double())[2].to(dt) if four else v
    # odd rows see their one slot; even ones 15 slots of zeros besides
    assert torch.allclose(out[1::2].float(), values[1::2].expand(-1, h, -1).float(), rtol=2.0 ** -7, atol=2.0 ** -20)
    for i in (0, 35000, b - 2):
        keys = torch.zeros(16, g, d, dtype=torch.float64, device="cuda")
        vals = keys.clone()
        keys[15], vals[15] = (_quantise(k[i].double())[2] if four else k[i].double()), values[i].double()
        _check_attention(out[i], None, q[i], keys, vals, d ** -0.5, dt, four)
    if four:
        all_ = ops.paged_attn_decode4(q, kp, vp, table, ln)
        assert torch.equal(all_[0::2], out[0::2])


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h, g, b, n", [(4, 2, 300, 700), (8, 1, 150, 1400), (16, 16, 30, 2500), (2, 2, 400, 90)])
def test_decode4_where_rows_fill_the_grid(dt, h, g, b, n):
    """A block or a small cluster per row, more rows than run at once."""
    from project_chronos_b200 import ops
    d = 64
    lens = [max(0, n - 7 * i) for i in range(b)]
    kp, vp, table, ln, rows = _cache4(lens, g, d, 16, 11)
    q = _rnd(12, b, h, d, dt=dt, scale=2.0)
    lse = torch.empty(b, h, device="cuda")
    out = ops.paged_attn_decode4(q, kp, vp, table, ln, lse=lse)
    ops.check_status(out.device)
    for i in sorted({0, 1, b // 2, b - 1}):
        _check_attention(out[i], lse[i], q[i], *rows[i], d ** -0.5, dt, True)


@gpu
@pytest.mark.parametrize("four", [False, True])
def test_calls_take_views(four):
    """A part of a wider page table, expanded queries, keys of one head read as several."""
    from project_chronos_b200 import ops
    h, g, d, size, dt = 8, 2, 64, 16, BF
    kp, vp, table, ln, rows = _cache4([100, 50], g, d, size, 3) if four else _cache16([100, 50], g, d, size, dt, 3)
    wide = torch.full((2, 3 * table.shape[1]), -1, dtype=torch.int32, device="cuda")
    part = wide[:, 2: 2 + table.shape[1]]
    part.copy_(table)
    q = _rnd(1, 1, 1, d, dt=dt).expand(2, h, d)
    pages = torch.arange(4, dtype=torch.int32, device="cuda").expand(2, g, 4).contiguous()
    got = ops.paged_attn_sparse(q, kp, vp, part, ln, pages)
    assert torch.equal(got, ops.paged_attn_sparse(q.contiguous(), kp, vp, table, ln, pages))
    bounds = torch.zeros(kp.shape[0], 2, g, d, dtype=dt, device="cuda")
    ops.paged_bounds(kp, bounds, part, ln, full=True)
    assert torch.equal(ops.paged_select(q, bounds, part, ln, size, 3), ops.paged_select(q.contiguous(), bounds, table, ln, size, 3))
    if four:
        assert torch.equal(ops.paged_attn_decode4(q, kp, vp, part, ln), ops.paged_attn_decode4(q.contiguous(), kp, vp, table, ln))
    cos, sin = _tables(200, d)
    one = _rnd(2, 2, 1, d, dt=dt)
    res = []
    for k, tab in ((one.expand(2, g, d), part), (one.expand(2, g, d).contiguous(), table)):
        a, b = kp.clone(), vp.clone()
        qq = ops.paged_append_rope(k, k, a, b, tab, ln, ln, cos[:1].expand(200, d), sin, q=q)
        res.append((a, b, qq))
    for x, y in zip(*res):
        assert torch.equal(x.nan_to_num(9.0) if x.is_floating_point() else x, y.nan_to_num(9.0) if y.is_floating_point() else y)
    ops.check_status(got.device)


@gpu
def test_two_streams_at_once():
    """Calls on two streams, each with its own workspace, keep out of each other's way."""
    from project_chronos_b200 import ops
    h, g, d, dt = 8, 2, 128, BF
    caches = [_cache4([9000 + 500 * i, 300], g, d, 16, 5 + i) for i in range(2)]
    qs = [_rnd(6 + i, 2, h, d, dt=dt, scale=2.0) for i in range(2)]
    bounds = [torch.zeros(c[0].shape[0], 2, g, d, dtype=dt, device="cuda") for c in caches]
    for c, b in zip(caches, bounds):
        ops.paged_bounds(c[0], b, c[2], c[3], full=True)
    def call(i):
        kp, vp, table, ln, _ = caches[i]
        pages = ops.paged_select(qs[i], bounds[i], table, ln, 16, 40, first=1, last=2)
        return ops.paged_attn_decode4(qs[i], kp, vp, table, ln), pages, ops.paged_attn_sparse(qs[i], kp, vp, table, ln, pages)
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[i]))


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
def test_append_rope_in_a_cache_that_evicts(dt):
    """Rotation on the way into a cache with running sums: positions go on counting tokens after an eviction."""
    from project_chronos_b200 import PagedCache, ops
    h, g, d, size = 4, 2, 64, 16
    c = PagedCache(2, 20, g, d, 10, "cuda", dt, page_size=size, track_weights=True)
    cos, sin = _tables(400, d)
    for b in range(2):
        c.reserve(b, 160)
    q, k, v = (_rnd(i, 200, x, d, dt=dt) for i, x in ((1, h), (2, g), (3, g)))
    c.append_rope(q[:180], k[:180], v[:180], cos, sin, cu_seqlens=_i32(0, 120, 180))
    c.attend(q[:2])
    c.evict(50, sinks=2, recent=8)
    assert c.lens.tolist() == [50, 50] and c.seen.tolist() == [120, 60]
    got = c.append_rope(q[180:182], k[180:182], v[180:182], cos, sin)
    ops.check_status(got.device)
    assert c.lens.tolist() == [51, 51] and c.seen.tolist() == [121, 61]
    for b, at in ((0, 120), (1, 60)):
        y, m = _rotate(q[180 + b: 181 + b].double(), cos[at: at + 1], sin[at: at + 1], 0)
        _near(got[b: b + 1], y, m, dt)
        y, m = _rotate(k[180 + b: 181 + b].double(), cos[at: at + 1], sin[at: at + 1], 0)
        _near(c.k_pages[c.page_table[b, 3].long(), 2][None], y, m, dt)
        assert bool((c.positions[b, :, 50] == at).all()) and bool((c.weights[b, :, 50] == 0).all())
    with pytest.raises(RuntimeError, match="page_bounds"):
        c.attend_sparse(q[:2], 2)


@gpu
def test_bounds_after_slots_were_given_up():
    """A draft is taken back: the bounds stay bounds, and are exact again from nothing."""
    from project_chronos_b200 import PagedCache, ops
    g, d, size, dt = 2, 64, 16, BF
    c = PagedCache(1, 8, g, d, 8, "cuda", dt, page_size=size, page_bounds=True)
    c.reserve(0, 100)
    k = _rnd(1, 60, g, d, dt=dt)
    c.append(k[:40], k[:40], _i32(0, 40))
    c.append(10 * k[40:44], k[40:44], _i32(0, 4))
    c.lens -= 3
    c.seen -= 3
    c.append(k[44:60], k[44:60], _i32(0, 16))
    rows = torch.cat([k[:40], 10 * k[40:41], k[44:60]])
    want = _bounds_of(rows, size)
    got = c.bounds[c.page_table[0, :4].long()]
    assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]]) and bool((got[2, 0] <= want[2, 0]).all()) and bool((got[2, 1] >= want[2, 1]).all())
    ops.paged_bounds(c.k_pages, c.bounds, c.page_table, c.lens, full=True)
    assert torch.equal(c.bounds[c.page_table[0, :4].long()], want)


@gpu
@pytest.mark.parametrize("four", [False, True])
def test_offsets_pass_32_bits(four):
    """Pages, rows and bounds that lie further apart than 32 bits count."""
    from project_chronos_b200 import ops
    h, g, d, size, dt = 8, 2, 128, 16, BF
    far = (1 << 31) + 64
    def rows(n, *heads):                                   # [n, heads, d] side by side, rows `far` elements apart
        store = torch.empty((n - 1) * far + sum(heads) * d, dtype=dt, device="cuda")
        return [store[sum(heads[:i]) * d:].as_strided((n, m, d), (far, d, 1)) for i, m in enumerate(heads)]
    if four:
        nbytes, apart = ops.packed_page_bytes(size, d), (1 << 32) - 16
        store = torch.empty(2 * apart + 2 * g * nbytes, dtype=torch.uint8, device="cuda")
        kp, vp = (store[i * g * nbytes:].as_strided((3, g, nbytes), (apart, nbytes, 1)) for i in range(2))
    else:
        store = torch.empty(2 * far + 2 * size * g * d, dtype=dt, device="cuda")
        kp, vp = (store[i * size * g * d:].as_strided((3, size, g, d), (far, g * d, d, 1)) for i in range(2))
    q, k, v = rows(2, h, g, g)
    for x, seed in ((q, 1), (k, 2), (v, 3)):
        x.copy_(_rnd(seed, *x.shape, dt=dt))
    table, ln = _i32(0, 1, 2, 0).view(2, 2), _i32(15, 15)
    first = _rnd(4, 30, g, d, dt=dt)
    ops.paged_append_rope(first, -first, kp, vp, table, _i32(0, 0), cu_seqlens=_i32(0, 15, 30))
    q_out, k_out, v_out = rows(2, h, g, g)
    ops.paged_append_rope(k, v, kp, vp, table, ln, q=q, q_out=q_out, lens_out=ln)
    assert torch.equal(q_out, q)
    ops.paged_gather(kp, vp, table, ln, _i32(0, 1, 2), k_out, v_out)
    ops.check_status(ln.device)
    def held(x):
        return _quantise(x.double())[2] if four else x.double()
    assert torch.equal(k_out.double(), held(k)) and torch.equal(v_out.double(), held(v))
    pages = torch.zeros(2, g, 1, dtype=torch.int32, device="cuda")
    out = rows(2, h)[0]
    ops.paged_attn_sparse(q, kp, vp, table, ln, pages, out=out)
    both = [out] + ([ops.paged_attn_decode4(q, kp, vp, table, ln)] if four else [])
    for i in range(2):
        keys, vals = (held(torch.cat([s * first[15 * i: 15 * i + 15], x[i: i + 1]])) for s, x in ((1, k), (-1, v)))
        for o in both:
            _check_attention(o[i], None, q[i], keys, vals, d ** -0.5, dt, four)
    bounds = torch.zeros(3, 2, g, d, dtype=dt, device="cuda")
    ops.paged_bounds(kp, bounds, table, ln, full=True)
    for i in range(2):
        keys = held(torch.cat([first[15 * i: 15 * i + 15], k[i: i + 1]])).to(dt)
        assert torch.equal(bounds[2 * i], _bounds_of(keys, size)[0])
    ops.check_status(ln.device)


@gpu
def test_select_among_bounds_that_pass_32_bits():
    from project_chronos_b200 import ops
    d, dt = 256, BF
    n = (1 << 31) // (2 * d) + 100                         # pages of a slot each
    kp = torch.zeros(n, 1, 1, d, dtype=dt, device="cuda")
    bounds = torch.zeros(n, 2, 1, d, dtype=dt, device="cuda")
    table, ln = _i32(n - 1, 5, n - 50, n - 2).view(1, 4), _i32(4)
    k = _rnd(1, 4, 1, d, dt=dt)
    kp[table[0].long(), 0] = k
    ops.paged_bounds(kp, bounds, table, ln, full=True)
    assert torch.equal(bounds[table[0].long()], torch.stack([k, k], 1))
    q = k[2].expand(1, 1, d)
    assert ops.paged_select(q, bounds, table, ln, 1, 2).view(-1).tolist() == [2, 3]
    ops.check_status(ln.device)
