"""The paged cache's further operators (include/chronos_paged4.h) at the edges of what they
take: bounds and queries that are not finite, rows at the ends of their type's range,
factors with many bits, windows over long rows, results that overlap inputs.

CPU: refusals.  GPU: against the definitions in 64 bits of test_paged4, with its tolerances.
"""
import ctypes
import math

import pytest
import torch

from test_paged4 import (BF, FP, HF, _attend, _cache4, _check_attention, _i32, _native_cache, _page_table, _quantise, _refuses, _rnd, _rotate,
                         _stored, _visible, gpu, lib)  # noqa: F401


# ---------------------------------------------------------------------------------------
# selection among bounds and queries that are not finite
# ---------------------------------------------------------------------------------------

def _literal(q, lo, hi, g, topk, first, last):
    """The pages of one token by the formula as it stands, head by head: q [H, D], lo and hi [m, G, D] -> [G, topk]."""
    m, h = lo.shape[0], q.shape[0]
    res = torch.full((g, topk), -1, dtype=torch.int32)
    for i in range(g):
        x = q[i * h // g: (i + 1) * h // g, None].double()
        score = torch.maximum(x * lo[:, i].double(), x * hi[:, i].double()).sum((0, 2)).tolist() if m else []

        def rank(j):
            if j < first or j >= m - last:
                return (0, 0.0, j)
            return (1, 0.0, j) if math.isnan(score[j]) else (2, -score[j], j)
        best = sorted(sorted(range(m), key=rank)[:topk])
        res[i, : len(best)] = torch.tensor(best, dtype=torch.int32)
    return res


def _odd_bounds(n, g, d, dt, seed):
    """Bounds of n pages, most of them ordinary; every tenth page has columns that are infinite on one side, on both,
    the same infinity twice, or no number."""
    bounds = _rnd(seed, n, 2, g, d).sort(dim=1).values
    kinds = [(-math.inf, None), (None, math.inf), (-math.inf, math.inf), (math.inf, math.inf), (-math.inf, -math.inf), (math.nan, math.nan),
             (-math.inf, None), (None, math.inf)]
    for i in range(0, n, 10):
        lo, hi = kinds[i // 10 % len(kinds)]
        columns = [(i * 7) % d] if i % 20 else [(i * 7) % d, (i * 3 + 1) % d, d - 1]
        for c in columns:
            if lo is not None:
                bounds[i, 0, :, c] = lo
            if hi is not None:
                bounds[i, 1, :, c] = hi
    return bounds.to(dt).contiguous()


@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("h, g, d", [(2, 2, 64), (8, 2, 128), (9, 1, 96), (16, 2, 256), (6, 3, 37)])
@pytest.mark.parametrize("queries", ["up", "down", "mixed", "some zero", "one infinite"])
@pytest.mark.parametrize("new", [None, [1, 9, 17]])
def test_select_among_bounds_that_are_not_finite(dt, h, g, d, queries, new):
    from project_chronos_b200 import ops
    size, topk, first, last, lens = 4, 60, 1, 2, [700, 1500, 1999]
    table, n = _page_table(3, 500, 1, 1)
    bounds = _odd_bounds(n, g, d, dt, 2)
    t = 3 if new is None else sum(new)
    q = _rnd(3, t, h, d)
    if queries == "up":
        q = q.abs() + 0.01
    elif queries == "down":
        q = -q.abs() - 0.01
    elif queries == "some zero":
        q = torch.where(torch.rand(q.shape, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") < 0.3, 0.0, q.abs() + 0.01)
        q[:, :, :4] = 0.0
    elif queries == "one infinite":
        q[::2, 0, 5] = math.inf
        q[1::2, h - 1, 6] = -math.inf
    q = q.to(dt)
    cu = None if new is None else torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    got = ops.paged_select(q, bounds, table, _i32(*lens), size, topk, first=first, last=last, cu_seqlens=cu)
    ops.check_status(got.device)
    row = 0
    for i in range(3):
        for j in range(1 if new is None else new[i]):
            at = lens[i] if new is None else lens[i] - new[i] + 1 + j
            m = -(-at // size)
            x = bounds[table[i, :m].long()]
            assert torch.equal(got[row].cpu(), _literal(q[row], x[:, 0], x[:, 1], g, topk, first, last)), (i, j)
            row += 1


@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("odd", [10, 20])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_an_infinite_bound_that_no_query_meets_changes_nothing(dt, odd, sign):
    """Two equal pages, one of them infinite on the side that the queries never take: the lower page goes first."""
    from project_chronos_b200 import ops
    h, g, d, m = 4, 2, 64, 60
    bounds = torch.zeros(m, 2, g, d, device="cuda")
    bounds[[10, 20]] = torch.tensor([-1.0, 1.0], device="cuda")[None, :, None, None]
    bounds[odd, 0 if sign > 0 else 1, :, 7] = -sign * math.inf
    q = sign * (_rnd(1, 1, h, d).abs() + 0.5)
    got = ops.paged_select(q.to(dt), bounds.to(dt), torch.arange(m, dtype=torch.int32, device="cuda").view(1, m), _i32(m), 1, 2)
    assert got[0].tolist() == [[10, 59]] * g


# ---------------------------------------------------------------------------------------
# 4-bit pages: rows at the ends of their type's range
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt, units", [(BF, (1.0, 1.0)), (BF, (0.5, 3.1)), (BF, (1e-30, 2.0 ** -126)), (HF, (1e-36, 2.0 ** -126)), (FP, (1.0, 1.0)),
                                       (FP, (0.37, 0.25)), (FP, (1e-30, 2.0 ** 126)), (BF, (2.0 ** 126, 1e37))])
@pytest.mark.parametrize("g, d, r", [(2, 128, 128), (3, 64, 32), (3, 37, 10)])
@pytest.mark.parametrize("packed", [False, True])
def test_4bit_pages_of_rows_that_pass_the_range_of_fp32(dt, units, g, d, r, packed):
    """Values whose rotation or quotient passes fp32 are finite all the same: the largest scale and code.  NaN and
    infinities stay what they are, blocks of zeros and small values too."""
    from project_chronos_b200 import ops
    size, t = 16, 24
    big = torch.finfo(dt).max
    def rows(seed):
        x = _rnd(seed, t, g, d).clamp(-2, 2) / 2 * big
        m = torch.arange(t, device="cuda") % 6
        x = torch.where((m == 1)[:, None, None], torch.sign(x) * big, x)
        x = torch.where((m == 2)[:, None, None], 0.0, x)
        x = torch.where((m == 3)[:, None, None], x * 1e-30, x)
        x = x.to(dt)
        x[4, 0, d // 2], x[10, 0, d // 3], x[16, 0, 0] = math.nan, math.inf, -math.inf
        return x
    k, v = rows(1), rows(2)
    a = torch.linspace(0.0, 6.0, 40 * r // 2, device="cuda", dtype=torch.float64).view(40, r // 2)
    cos, sin = torch.cat([a.cos(), a.cos()], 1).float(), torch.cat([a.sin(), a.sin()], 1).float()
    b = 2 if packed else t
    new = [9, 15] if packed else [1] * t
    table, n = _page_table(b, 2, 1, 3)
    kp, vp = (torch.zeros(n, g, ops.packed_page_bytes(size, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    cu = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32) if packed else None
    ops.paged_append_rope(k, v, kp, vp, table, _i32(*[0] * b), _i32(*[5] * b), cos, sin, cu_seqlens=cu, k_scale=units[0], v_scale=units[1])
    ops.check_status(kp.device)
    at = 0
    for i, m in enumerate(new):
        part = slice(at, at + m)
        turned, _ = _rotate(k[part].double(), cos[5: 5 + m], sin[5: 5 + m], 0)
        for pages, x, unit in ((kp, turned, units[0]), (vp, v[part].double(), units[1])):
            code, scale, _ = _quantise(x, unit)
            code_, scale_, _ = _stored(pages, table[i], d, size, torch.arange(m, device="cuda"))
            assert torch.equal(scale_[..., : scale.shape[-1]], scale)
            assert torch.equal(code_[..., :d], code)
        at += m


# ---------------------------------------------------------------------------------------
# factors
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("factor", [1e-45, 1e-39, 1.17e-38, 2.0 ** -126 * (1 - 2.0 ** -23), 2.0 ** 126 * (1 + 2.0 ** -23), 3e38])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_factors_without_a_reciprocal_are_refused(lib, factor, which):  # noqa: F811
    from project_chronos_b200 import _native as N
    one = {**dict(k_scale=1.0, v_scale=1.0), which: factor}
    c = _native_cache(N)
    _refuses(lib, "append_rope", N.ChronosPagedRopeArgs(cache=c, num_tokens=2, packed=1, **one), which.encode())
    _refuses(lib, "gather", N.ChronosPagedGatherArgs(cache=c, num_tokens=2, packed=1, **one), which.encode())
    _refuses(lib, "decode4", N.ChronosPagedDecode4Args(cache=c, heads=2, scale=1.0, **one), which.encode(), workspace=True)
    _refuses(lib, "sparse", N.ChronosPagedSparseArgs(cache=c, heads=2, scale=1.0, num_tokens=2, packed=1, **one), which.encode())
    if which == "k_scale":
        _refuses(lib, "bounds", N.ChronosPagedBoundsArgs(cache=c, packed=1, k_scale=factor), b"k_scale")


@pytest.mark.parametrize("factor", [2.0 ** -126, 2.0 ** 126, 0.37])
def test_factors_with_a_reciprocal_are_taken(lib, factor):  # noqa: F811
    from project_chronos_b200 import _native as N
    a = N.ChronosPagedDecode4Args(cache=_native_cache(N, batch=0), heads=2, scale=1.0, k_scale=factor, v_scale=factor)
    assert lib.chronos_paged_decode4(ctypes.byref(a), None) == N.CHRONOS_OK


@pytest.mark.parametrize("scale, factor", [(1e-3, 2.0 ** -126), (4.0, 2.0 ** 126), (1e-30, 1e-30)])
def test_scores_without_a_factor_in_fp32_are_refused(lib, scale, factor):  # noqa: F811
    from project_chronos_b200 import _native as N
    one = dict(heads=2, scale=scale, k_scale=factor, v_scale=1.0)
    _refuses(lib, "decode4", N.ChronosPagedDecode4Args(cache=_native_cache(N), **one), b"scale", workspace=True)
    _refuses(lib, "sparse", N.ChronosPagedSparseArgs(cache=_native_cache(N), num_tokens=2, packed=1, **one), b"scale")


# ---------------------------------------------------------------------------------------
# bounds of 4-bit pages
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("factor", [0.37, 3.1, 1.0, 1e-6, 40.0])
@pytest.mark.parametrize("g, d, size", [(2, 128, 16), (1, 37, 32)])
def test_no_key_of_a_4bit_page_lies_outside_its_bounds(dt, factor, g, d, size):
    """A factor with many bits: the keys have more than the bounds' type.  The bounds lie less than a step outside."""
    from project_chronos_b200 import PagedCache, ops
    c = PagedCache(2, 20, g, d, 8, "cuda", dt, page_size=size, four_bit=True, page_bounds=True, k_scale=factor)
    for b in range(2):
        c.reserve(b, 100)
    x = factor * _rnd(1, 83, g, d)
    x[3::7] *= 400.0
    x = x.to(dt)
    c.append(x[:70], x[:70], _i32(0, 50, 70))
    for i in range(70, 83):
        c.append(x[i: i + 1], x[i: i + 1], _i32(0, 0, 1))
    ops.check_status(c.lens.device)
    lens = c.lens.tolist()
    assert lens == [50, 33]
    def check():
        for b in range(2):
            key = _stored(c.k_pages, c.page_table[b], d, size, torch.arange(lens[b], device="cuda"))[2] * float(torch.tensor(factor))
            for j, part in enumerate(key.split(size)):
                low, high = part.amin(0), part.amax(0)
                got = c.bounds[c.page_table[b, j].long()].double()
                assert bool((got[0] <= low).all()) and bool((got[1] >= high).all())
                step = lambda v: torch.finfo(dt).eps * v.abs() + (2.0 ** -24 if dt == HF else 0.0)  # noqa: E731
                near = high.abs() < torch.finfo(dt).max
                assert bool((low - got[0] <= step(low))[low.abs() < torch.finfo(dt).max].all()) and bool((got[1] - high <= step(high))[near].all())
    check()
    c.bounds.fill_(math.nan)
    ops.paged_bounds(c.k_pages, c.bounds, c.page_table, c.lens, full=True, k_scale=factor)
    check()


# ---------------------------------------------------------------------------------------
# 4-bit attention: windows and first tokens over long rows, heads of 256
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("h, g, d", [(8, 2, 64), (24, 1, 128), (4, 2, 128), (12, 2, 256), (20, 1, 256), (10, 2, 80)])
@pytest.mark.parametrize("lens", [[20011], [6001, 3, 0, 9000, 4100]])
@pytest.mark.parametrize("window, sinks", [(0, 0), (4097, 0), (5000, 17), (4999, 300), (4096, 4096)])
def test_decode4_windows_over_long_rows(lib, dt, h, g, d, lens, window, sinks):  # noqa: F811
    """Rows that are cut evenly over the blocks (the calls that need a workspace)."""
    from project_chronos_b200 import _native as N
    from project_chronos_b200 import ops
    kp, vp, table, ln, rows = _cache4(lens, g, d, 16, h + d)
    shape = N.ChronosPagedCache(batch=len(lens), kv_heads=g, head_dim=d, dtype=N.DTYPE_BF16 if dt == BF else N.DTYPE_FP32, num_pages=kp.shape[0],
                                page_size=16, table_width=table.shape[1])
    a = N.ChronosPagedDecode4Args(cache=shape, heads=h, window=window, sinks=sinks, scale=1.0, k_scale=1.0, v_scale=1.0)
    assert lib.chronos_paged_decode4_workspace(ctypes.byref(a)) > 0
    q = _rnd(6, len(lens), h, d, dt=dt, scale=2.0)
    lse = torch.empty(len(lens), h, device="cuda")
    out = ops.paged_attn_decode4(q, kp, vp, table, ln, window=window, sinks=sinks, lse=lse)
    ops.check_status(out.device)
    for b, (k, v) in enumerate(rows):
        seen = _visible(lens[b], window, sinks)
        _check_attention(out[b], lse[b], q[b], k[seen], v[seen], d ** -0.5, dt, True)
    assert torch.equal(out, ops.paged_attn_decode4(q, kp, vp, table, ln, window=window, sinks=sinks))
    over = q.clone()
    assert ops.paged_attn_decode4(over, kp, vp, table, ln, window=window, sinks=sinks, out=over) is over and torch.equal(over, out)


# ---------------------------------------------------------------------------------------
# results that overlap what a call reads
# ---------------------------------------------------------------------------------------

KP, VP, TABLE, LENS, Q, OUT, LSE, CU, LIST, BOUNDS = (i << 20 for i in range(1, 11))


def _full_cache(N, **kw):
    """2 sequences of 2 heads of 16 columns in 4 pages of 16 slots; 4-bit pages of 16 * 36 bytes a head."""
    return _native_cache(N, **{**dict(k_pages=KP, v_pages=VP, k_page_stride=1152, k_slot_stride=32, k_head_stride=576, v_page_stride=1152,
                                      v_slot_stride=32, v_head_stride=576, page_table=TABLE, page_table_stride=2, lens=LENS), **kw})


@pytest.mark.parametrize("change", [
    dict(out=Q + 64), dict(out=Q, out_row_stride=128), dict(out=KP + 4 * 1152 - 16), dict(out=VP), dict(out=LENS - 64), dict(out=TABLE), dict(lse=OUT),
    dict(lse=Q + 4), dict(lse=LENS + 4), dict(lse=KP), dict(q=OUT + 254)])
def test_attention_results_that_overlap_are_refused(lib, change):  # noqa: F811
    from project_chronos_b200 import _native as N
    f = dict(heads=4, scale=0.25, k_scale=1.0, v_scale=1.0, q=Q, q_row_stride=64, q_head_stride=16, out=OUT, out_row_stride=64, out_head_stride=16, lse=LSE)
    _refuses(lib, "decode4", N.ChronosPagedDecode4Args(cache=_full_cache(N), **{**f, **change}), b"overlap")
    f.update(num_tokens=2, topk=2, pages=LIST, packed=1)
    _refuses(lib, "sparse", N.ChronosPagedSparseArgs(cache=_full_cache(N), **{**f, **change}), b"overlap")


@pytest.mark.parametrize("change", [dict(out=LIST), dict(lse=LIST + 12), dict(out=CU - 250), dict(lse=CU + 8)])
def test_sparse_results_over_lists_and_offsets_are_refused(lib, change):  # noqa: F811
    from project_chronos_b200 import _native as N
    f = dict(heads=4, scale=0.25, k_scale=1.0, v_scale=1.0, q=Q, q_row_stride=64, q_head_stride=16, out=OUT, out_row_stride=64, out_head_stride=16, lse=LSE,
             num_tokens=2, topk=2, pages=LIST, cu_seqlens=CU)
    _refuses(lib, "sparse", N.ChronosPagedSparseArgs(cache=_full_cache(N), **{**f, **change}), b"overlap")


@pytest.mark.parametrize("pages", [TABLE, LENS + 4, Q, BOUNDS + 256, CU])
def test_selections_that_overlap_are_refused(lib, pages):  # noqa: F811
    from project_chronos_b200 import _native as N
    f = dict(heads=4, topk=3, last=1, num_tokens=2, q=Q, q_row_stride=64, q_head_stride=16, bounds=BOUNDS, cu_seqlens=CU, pages=pages)
    _refuses(lib, "select", N.ChronosPagedSelectArgs(cache=_full_cache(N), **f), b"overlap")


@pytest.mark.parametrize("bounds", [TABLE - 500, LENS, KP, KP + 3 * 1152 * 2, CU])
def test_bounds_that_overlap_are_refused(lib, bounds):  # noqa: F811
    from project_chronos_b200 import _native as N
    _refuses(lib, "bounds", N.ChronosPagedBoundsArgs(cache=_full_cache(N), num_tokens=2, bounds=bounds, cu_seqlens=CU), b"overlap")


@pytest.mark.parametrize("change", [
    dict(q_out=KP), dict(q_out=VP + 4 * 1152 - 32), dict(k_out=KP + 1152), dict(k_out=TABLE), dict(q_out=LENS), dict(q_out=11 << 20), dict(k_out=12 << 20),
    dict(lens_out=CU), dict(lens_out=TABLE), dict(seen_out=TABLE + 8), dict(seen_out=OUT), dict(q_out=13 << 20)])
def test_append_results_that_overlap_are_refused(lib, change):  # noqa: F811
    from project_chronos_b200 import _native as N
    rows = {f"{x}_{y}_stride": s for x in ("k", "v", "q", "q_out", "k_out") for y, s in (("row", 64), ("head", 16))}
    f = dict(num_tokens=2, heads=4, rope_dim=4, table_len=10, k=14 << 20, v=15 << 20, q=Q, q_out=OUT, cos=11 << 20, sin=12 << 20, cos_row_stride=4,
             sin_row_stride=4, cu_seqlens=CU, seen=13 << 20, packed=1, k_scale=1.0, v_scale=1.0, **rows)
    _refuses(lib, "append_rope", N.ChronosPagedRopeArgs(cache=_full_cache(N), **{**f, **change}), b"overlap")


@gpu
@pytest.mark.parametrize("four", [False, True])
def test_results_beside_their_inputs_are_taken(four):
    """In q itself, in other columns of q's array, and with one row in q's place with another stride."""
    from project_chronos_b200 import ops
    h, g, d, size = 4, 2, 64, 16
    kp, vp, table, ln, _ = _cache4([100, 50], g, d, size, 3)
    if not four:
        kp, vp = (torch.randn(kp.shape[0], size, g, d, device="cuda").to(BF) for _ in range(2))
    pages = torch.arange(3, dtype=torch.int32, device="cuda").expand(2, g, 3).contiguous()
    both = _rnd(4, 2, 2 * h, d, dt=BF)
    q = both[:, :h]
    calls = [lambda q, n=2, **kw: ops.paged_attn_sparse(q, kp, vp, table[:n], ln[:n], pages[:n], **kw)]
    if four:
        calls.append(lambda q, n=2, **kw: ops.paged_attn_decode4(q, kp, vp, table[:n], ln[:n], **kw))
    for call in calls:
        want = call(q)
        ops.check_status(want.device)
        assert torch.equal(call(q, out=both[:, h:]), want) and torch.equal(both[:, h:], want)
        over = both.clone()
        assert torch.equal(call(over[:, :h], out=over[:, :h]), want)
        one = q[:1].clone()
        assert torch.equal(call(one, 1, out=one.as_strided((1, h, d), (7 * d, d, 1))), want[:1])
        with pytest.raises(RuntimeError, match="overlap"):
            call(both[:, :h], out=both[:, 1: h + 1])
        with pytest.raises(RuntimeError, match="overlap"):
            call(q, lse=kp.view(-1).view(torch.float32)[: 2 * h].view(2, h))
    bounds = torch.zeros(kp.shape[0], 2, g, d, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        ops.paged_select(q, bounds, table, ln, size, 2, out=table.view(-1)[: 2 * g * 2].view(2, g, 2))


# ---------------------------------------------------------------------------------------
# the native module
# ---------------------------------------------------------------------------------------

def test_a_native_module_of_another_torch_or_python_is_built_again_and_not_loaded(lib, monkeypatch):  # noqa: F811
    from project_chronos_b200 import build, ops
    assert build.binding_fits(False) and not build.needs_binding()
    monkeypatch.setattr(ops, "_native_calls", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert not build.binding_fits(False) and build.needs_binding()
    with pytest.raises(RuntimeError, match="another Python or torch"):
        ops.paged_gather(*[torch.zeros(1)] * 7)
    monkeypatch.undo()
    monkeypatch.setattr(ops, "_native_calls", None)
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399")
    assert build.needs_binding()
    monkeypatch.undo()
    assert build.binding_fits(False)


def test_a_native_module_without_a_record_is_built_again(lib, monkeypatch, tmp_path):  # noqa: F811
    from project_chronos_b200 import build
    monkeypatch.setattr(build, "BINDING_STAMP", str(tmp_path / "none"))
    assert build.needs_binding() and build.binding_fits(True)


# ---------------------------------------------------------------------------------------
# weights of selected pages
# ---------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("h, d", [(8, 128), (24, 64), (8, 256)])
def test_fp16_weights_of_selected_pages_keep_more_than_a_half(four, h, d):
    """Two slots with values 6 and -6 and nearly equal scores: what is left is the difference of two weights.  Each is off
    by 2^-22 in two halves (2^-11 in one), the rest is the fp32 part of test_paged4's tolerance."""
    from project_chronos_b200 import ops
    g, size, dt = 2, 16, HF
    k = torch.zeros(2, g, d, dtype=dt, device="cuda")
    k[:, :, 1], k[0, :, 0] = 6.0, 1.0                      # 4 bits hold them
    v = torch.full_like(k, 6.0)
    v[1] = -6.0
    table = _i32(0).view(1, 1)
    if four:
        kp, vp = (torch.zeros(1, g, ops.packed_page_bytes(size, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        kp, vp = (torch.zeros(1, size, g, d, dtype=dt, device="cuda") for _ in range(2))
    ops.paged_append_rope(k, v, kp, vp, table, _i32(0), cu_seqlens=_i32(0, 2))
    q = torch.zeros(1, h, d, dtype=dt, device="cuda")
    q[0, :, 0] = torch.linspace(1e-4, 1e-2, h, device="cuda")
    out = ops.paged_attn_sparse(q, kp, vp, table, _i32(2), torch.zeros(1, g, 1, dtype=torch.int32, device="cuda"), scale=1.0)[0].double()
    ops.check_status(kp.device)
    ref, _, a, s, s2 = _attend(q[0], k, v, 1.0)
    f = d * 2.0 ** -23 * s + 2 * 2.0 ** -24 + 2.0 ** -20 + (2.0 ** -28 * s2 if four else 0.0)
    tol = torch.finfo(dt).eps / 2 * ref.abs() + (f[:, None] + 2 * 2.0 ** -23 + 2.0 ** -21) * a + 2.0 ** -25
    err = (out - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of the tolerance"


@gpu
def test_results_that_no_memory_holds_raise_as_torch_does():
    """A selection of 2^31 - 1 pages for 64 heads: 550 GB."""
    from project_chronos_b200 import ops
    q, bounds = _rnd(1, 4, 16, 64, dt=BF), torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda")
    table, ln = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), _i32(1, 1, 1, 1)
    with pytest.raises(torch.OutOfMemoryError):
        ops.paged_select(q, bounds, table, ln, 16, 2 ** 31 - 1)
    assert ops.paged_select(q, bounds, table, ln, 16, 2).shape == (4, 16, 2)
    ops.check_status(q.device)
