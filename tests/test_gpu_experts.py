"""Expert routing, the expert FFN and the sandwich norm on the B200, against
64-bit computations of the same formulas.

Tolerances.  u is half a step of the stored 16-bit type (finfo.eps / 2).
 * Routing: indices, offsets and slots are equal.  Weights: expf within 2 ulp,
   a sum of up to 512 terms (21 roundings deep), divisions: 32 * 2^-24 relative.
 * Products: fp16/bf16 products are exact in fp32; a sum over K in steps of 16
   has at most K/16 + 16 roundings of 2^-23 of sum |a w|; the hidden layer and
   each expert's output are rounded once (u); GELU is within 5e-7.  Bounds are
   carried through W_out elementwise, which no wrong expert, row or bias stays
   inside of.  The bound ignores that rounding errors cancel, so the rms of the
   error is held to 4 u of the output's rms too (three independent roundings of
   at most u / sqrt(3) rms make u).
 * Norms: a row's sums are at most 75 roundings deep (64 columns per thread,
   then a tree): 128 * 2^-24 of the largest normalised value, plus u |y|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0**-24


@pytest.fixture(autouse=True)
def _sync_check(cuda_pkg):
    prev = cuda_pkg._lib.set_sync_check(True)
    yield
    cuda_pkg._lib.set_sync_check(prev)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


# ---- routing -------------------------------------------------------------------
def _ref_route(logits, k, scoring, bias=None, groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0, live=None):
    x = logits.double().cpu().numpy()
    T, E = x.shape
    shut = ~(x > -np.inf)
    xs = np.where(shut, -np.inf, x)
    with np.errstate(all="ignore"):
        if scoring == "softmax":
            m = np.where(shut.all(1, keepdims=True), 0.0, xs.max(1, keepdims=True))
            p = np.exp(xs - m)
            z = p.sum(1, keepdims=True)
            s = np.where(z > 0, p / np.where(z > 0, z, 1), 0.0)
        else:
            s = np.exp(-np.logaddexp(0.0, -xs))
    v = s + (0.0 if bias is None else bias.double().cpu().numpy()[None])
    if bias is None and group_top == 1:
        v = xs.copy()  # the same order, without underflow
    v[shut] = -np.inf
    if groups > 1:
        per = E // groups
        g = -np.sort(-v.reshape(T, groups, per), axis=2)[:, :, :group_top]
        st = np.where(np.isneginf(g), 0.0, g).sum(2)
        st[shut.reshape(T, groups, per).all(2)] = -np.inf
        keep = np.zeros((T, groups), bool)
        np.put_along_axis(keep, np.argsort(-st, 1, kind="stable")[:, :top_groups], True, 1)
        v[~np.repeat(keep, per, 1)] = -np.inf
    idx = np.argsort(-v, 1, kind="stable")[:, :k]
    none = np.isneginf(np.take_along_axis(v, idx, 1))
    w = np.where(none, 0.0, np.take_along_axis(s, idx, 1))
    if renorm:
        tot = w.sum(1, keepdims=True)
        w = np.where(tot > 0, w / np.where(tot > 0, tot, 1), 0.0)
    idx = np.where(none, -1, idx)
    w = w * scale
    if live is not None:
        idx[live:] = -1
        w[live:] = 0.0
    return idx, w


def _ref_plan(idx, E):
    T, k = idx.shape
    flat = idx.reshape(-1)
    taken = np.flatnonzero(flat >= 0)
    slots = taken[np.argsort(flat[taken], kind="stable")]
    slot_row = np.full(T * k, -1)
    slot_row[: slots.size] = slots // k
    row_slot = np.full(T * k, -1)
    row_slot[slots] = np.arange(slots.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[taken], minlength=E))])
    return offsets, slot_row, row_slot.reshape(T, k)


def _check_plan(r, idx, E):
    offsets, slot_row, row_slot = _ref_plan(idx, E)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.slot_row.cpu().numpy(), slot_row)
    assert np.array_equal(r.row_slot.cpu().numpy(), row_slot)


def _check_route(cuda_pkg, logits, k, scoring="softmax", live=None, **kw):
    names = {"groups": "num_groups", "group_top": "group_score_top", "renorm": "renormalize", "scale": "weight_scale"}
    count = None if live is None else torch.tensor([live], dtype=torch.int32, device=DEV)
    r = cuda_pkg.kernels.route_experts(logits, k, scoring=scoring, row_count=count,
                                       **{names.get(n, n): v for n, v in kw.items()})
    idx, w = _ref_route(logits, k, scoring, live=live, **kw)
    assert np.array_equal(r.experts.cpu().numpy(), idx)
    err = np.abs(r.weights.double().cpu().numpy() - w)
    assert (err <= 32 * U32 * w + 1e-37).all(), err.max()
    _check_plan(r, idx, logits.shape[1])
    return r


# One row, one CTA (up to 32 rows), a chunk per CTA, many rows per chunk; every
# number of experts per lane and odd ones; E = 1; top_k = E.
@pytest.mark.parametrize("rows,E,k", [(1, 8, 2), (1, 1, 1), (7, 5, 5), (32, 32, 32), (33, 33, 4), (64, 64, 6),
                                      (257, 100, 8), (5000, 128, 1), (1001, 256, 8), (300, 512, 16), (20011, 7, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route(cuda_pkg, rows, E, k, dtype, scoring):
    g = _gen(rows * 31 + E)
    logits = _randn(g, rows, E, std=2.0).to(dtype)
    _check_route(cuda_pkg, logits, k, scoring)
    _check_route(cuda_pkg, logits, k, scoring, renorm=False, scale=2.5)


@pytest.mark.parametrize("rows,E,k,groups,top", [(1, 8, 2, 4, 1), (40, 64, 6, 8, 3), (3000, 256, 8, 8, 4),
                                                 (500, 60, 5, 5, 2), (500, 66, 3, 2, 1), (100, 32, 2, 32, 2),
                                                 (200, 512, 8, 16, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_groups_and_bias(cuda_pkg, rows, E, k, groups, top, scoring, biased):
    g = _gen(rows + E)
    logits = _randn(g, rows, E, std=1.5)
    logits[torch.rand(rows, E, generator=g, device=DEV) < 0.05] = -math.inf
    bias = _randn(g, E, std=0.05) if biased else None
    for group_top in ([1, 2] if E // groups > 1 else [1]):
        _check_route(cuda_pkg, logits, k, scoring, bias=bias, groups=groups, top_groups=top, group_top=group_top)


# Tiles whose last rows do not fill their warps, in every chunk but one.
@pytest.mark.parametrize("rows", [9473, 90077])
def test_route_groups_partial_tiles(cuda_pkg, rows):
    g = _gen(rows)
    logits = _randn(g, rows, 64, std=1.5)
    logits[torch.rand(rows, generator=g, device=DEV) < 0.02] = -math.inf
    bias = _randn(g, 64, std=0.05)
    for _ in range(3):
        _check_route(cuda_pkg, logits, 6, "sigmoid", bias=bias, groups=8, top_groups=3, group_top=2, scale=2.5)
    _check_route(cuda_pkg, logits, 4, "softmax", groups=4, top_groups=1)


@pytest.mark.parametrize("E,groups,top", [(64, 1, 1), (200, 1, 1), (64, 8, 3)])
def test_route_values_closer_than_fp32(cuda_pkg, E, groups, top):
    """The bias nearly cancels the score: all values lie within 1e-7 and only
    64 bits tell their order."""
    g = _gen(5)
    base = _randn(g, 1, E, dtype=torch.bfloat16)
    logits = base.repeat(300, 1)
    swap = torch.randint(0, E, (300,), generator=g, device=DEV)
    logits[torch.arange(300, device=DEV), swap] += 1.0
    bias = (0.75 - torch.sigmoid(base.double()[0])).float()
    _check_route(cuda_pkg, logits, 6, "sigmoid", bias=bias, groups=groups, top_groups=top, group_top=2)


def test_route_ties_take_the_lowest_index(cuda_pkg):
    logits = torch.zeros(50, 96, device=DEV)
    logits[:, 40] = -0.0
    r = _check_route(cuda_pkg, logits, 5)
    assert torch.equal(r.experts[0].cpu(), torch.arange(5, dtype=torch.int32))
    _check_route(cuda_pkg, logits, 5, "sigmoid", bias=torch.zeros(96, device=DEV), groups=4, top_groups=2, group_top=2)
    coarse = torch.randint(-2, 3, (777, 64), generator=_gen(1), device=DEV).half()
    _check_route(cuda_pkg, coarse, 8)
    _check_route(cuda_pkg, coarse, 8, "softmax", bias=torch.zeros(64, device=DEV), renorm=False)


def test_route_closed_experts_and_rows(cuda_pkg):
    g = _gen(9)
    logits = _randn(g, 200, 24)
    logits[3] = -math.inf  # no expert
    logits[4, 1:] = -math.inf  # one expert
    logits[5, 12:] = -math.inf
    logits[:, 7] = -math.inf  # closed to every row
    for scoring in ("softmax", "sigmoid"):
        for renorm in (False, True):
            r = _check_route(cuda_pkg, logits, 4, scoring, renorm=renorm)
            assert (r.experts[3] == -1).all() and (r.weights[3] == 0).all()
            assert r.experts[4].tolist() == [0, -1, -1, -1]
        _check_route(cuda_pkg, logits, 4, scoring, bias=_randn(g, 24), groups=4, top_groups=2, group_top=2)
    _check_route(cuda_pkg, torch.full((70, 16), -math.inf, device=DEV), 3)


def test_route_far_logits(cuda_pkg):
    """Scores that underflow fp32 while their ratios do not, and the type's lowest value."""
    g = _gen(11)
    logits = _randn(g, 64, 32) * 0.25 - 150.0
    r = cuda_pkg.kernels.route_experts(logits, 4, scoring="sigmoid")
    idx, w = _ref_route(logits, 4, "sigmoid")
    assert np.array_equal(r.experts.cpu().numpy(), idx)
    # exp(x - max) of exact differences
    assert np.abs(r.weights.double().cpu().numpy() - w).max() <= 32 * U32
    low = torch.full((10, 16), torch.finfo(torch.float32).min, device=DEV)
    low[:, 3] = 1.0
    _check_route(cuda_pkg, low, 2)
    _check_route(cuda_pkg, logits + 400.0, 4, "sigmoid", renorm=False)


def test_route_past_32_bit_offsets(cuda_pkg):
    """rows * experts above 2^31 elements."""
    rows, E = 8_400_000, 256
    logits = torch.empty(rows, E, device=DEV, dtype=torch.bfloat16)
    g = _gen(21)
    for c in logits.split(600_000):
        c.normal_(generator=g)
    r = cuda_pkg.kernels.route_experts(logits, 1, renormalize=False, scoring="sigmoid")
    e = torch.arange(E, device=DEV, dtype=torch.int32)
    for lo in range(0, rows, 600_000):
        c = logits[lo : lo + 600_000]
        first = torch.where(c == c.amax(1, keepdim=True), e, E).amin(1)
        assert torch.equal(r.experts[lo : lo + 600_000, 0], first)
    flat = r.experts.flatten().long()
    assert torch.equal(r.offsets[1:].long(), torch.bincount(flat, minlength=E).cumsum(0))
    assert torch.equal(r.slot_row.long(), flat.sort(stable=True)[1])


@pytest.mark.parametrize("kw", [dict(num_groups=3), dict(num_groups=0), dict(num_groups=64, top_groups=1),
                                dict(num_groups=4, top_groups=5), dict(num_groups=4, top_groups=0),
                                dict(num_groups=16, top_groups=1), dict(num_groups=4, top_groups=2, group_score_top=3)])
def test_route_refuses_groups(cuda_pkg, kw):
    with pytest.raises(cuda_pkg._lib.TJError, match="group"):
        cuda_pkg.kernels.route_experts(torch.zeros(4, 64, device=DEV), 6, **kw)


def test_gemm_refuses_widths(cuda_pkg):
    k = cuda_pkg.kernels
    r = k.route_experts(torch.zeros(4, 2, device=DEV), 1)
    with pytest.raises(cuda_pkg._lib.TJError, match="multiples of 8"):
        k.gemm_experts(torch.zeros(4, 12, dtype=torch.float16, device=DEV), torch.zeros(2, 8, 12, dtype=torch.float16, device=DEV),
                       None, r, gather=True)
    with pytest.raises(cuda_pkg._lib.TJError, match="multiples of 8"):
        k.expert_ffn(torch.zeros(4, 16, dtype=torch.float16, device=DEV), torch.zeros(2, 12, 16, dtype=torch.float16, device=DEV),
                     None, torch.zeros(2, 16, 12, dtype=torch.float16, device=DEV), None, r)
    odd = torch.zeros(4 * 16 + 1, dtype=torch.float16, device=DEV)[1:].view(4, 16)
    with pytest.raises(cuda_pkg._lib.TJError, match="aligned"):
        k.gemm_experts(odd, torch.zeros(2, 8, 16, dtype=torch.float16, device=DEV), None, r, gather=True)


def test_route_nan_rows(cuda_pkg):
    logits = _randn(_gen(2), 100, 40)
    clean = cuda_pkg.kernels.route_experts(logits, 3)
    bad = logits.clone()
    bad[10, 5] = math.nan
    bad[20] = math.nan
    bad[30, 7] = math.inf
    for kw in ({}, {"bias": torch.zeros(40, device=DEV), "num_groups": 4, "top_groups": 2, "group_score_top": 2}):
        r = cuda_pkg.kernels.route_experts(bad, 3, **kw)
        for row in (10, 20, 30):
            assert torch.isnan(r.weights[row]).all()
        assert ((r.experts >= -1) & (r.experts < 40)).all()
        assert (r.experts[10] != 5).all() and (r.experts[20] == -1).all()
        _check_plan(r, r.experts.cpu().numpy(), 40)
    ok = [i for i in range(100) if i not in (10, 20, 30)]
    r = cuda_pkg.kernels.route_experts(bad, 3)
    assert torch.equal(r.experts[ok], clean.experts[ok]) and torch.equal(r.weights[ok], clean.weights[ok])


@pytest.mark.parametrize("rows,live", [(20, 0), (20, 13), (20, 99), (3000, 0), (3000, 1), (3000, 2999)])
def test_route_row_count(cuda_pkg, rows, live):
    logits = _randn(_gen(rows), rows, 48)
    logits[min(live, rows) :] = math.nan  # rows behind the last are not read
    _check_route(cuda_pkg, logits.nan_to_num(0.0), 4, live=live)
    r = cuda_pkg.kernels.route_experts(logits, 4, row_count=torch.tensor([live], dtype=torch.int32, device=DEV))
    assert (r.experts[live:] == -1).all() and (r.weights[live:] == 0).all()


@pytest.mark.parametrize("rows,k,E", [(1, 1, 1), (30, 4, 9), (5000, 3, 512), (40000, 2, 6)])
def test_expert_plan(cuda_pkg, rows, k, E):
    g = _gen(rows)
    idx = torch.randint(-1, E, (rows, k), generator=g, device=DEV, dtype=torch.int32)
    idx[0] = 0  # the same expert twice
    idx[rows // 2 :, 0] = E - 1  # one busy expert
    r = cuda_pkg.kernels.expert_plan(idx, torch.ones(rows, k, device=DEV), E)
    _check_plan(r, idx.cpu().numpy(), E)


def test_expert_plan_reports_bad_index(cuda_pkg):
    L = cuda_pkg._lib
    idx = torch.randint(0, 8, (300, 2), device=DEV, dtype=torch.int32)
    idx[200, 1] = 8
    with pytest.raises(L.TJError, match="outside"):
        cuda_pkg.kernels.expert_plan(idx, torch.ones(300, 2, device=DEV), 8)
    L.set_sync_check(False)
    r = cuda_pkg.kernels.expert_plan(idx, torch.ones(300, 2, device=DEV), 8)
    with pytest.raises(L.TJError):
        L.device_status(torch.cuda.current_stream().cuda_stream)
    idx[200, 1] = -1
    _check_plan(r, idx.cpu().numpy(), 8)


def test_route_empty(cuda_pkg):
    k = cuda_pkg.kernels
    r = k.route_experts(torch.empty(0, 8, device=DEV), 2)
    assert r.experts.shape == (0, 2) and (r.offsets == 0).all()
    r = k.expert_plan(torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, device=DEV), 8)
    assert (r.offsets == 0).all()
    w = torch.zeros(8, 16, 16, dtype=torch.float16, device=DEV)
    out = k.expert_ffn(torch.empty(0, 16, dtype=torch.float16, device=DEV), w, None, w, None, r)
    assert out.shape == (0, 16)
    y = k.gemm_experts(torch.empty(0, 16, dtype=torch.float16, device=DEV), w, None, r, gather=True)
    assert k.expert_combine(y, r).shape == (0, 16)


# ---- expert FFN ----------------------------------------------------------------
def _weights(g, E, N, K, dtype, std=None):
    return _randn(g, E, N, K, dtype=dtype, std=K**-0.5 if std is None else std)


def _acc_bound(K):
    return (K / 16 + 16) * 2.0**-23


def _ref_gemm(a, w, b, slot_row, offsets, gather, gelu):
    """Slots' products in 64 bits and the bound on the kernel's error before storing."""
    n = int(offsets[-1])
    rows = slot_row[:n].long()
    src = a[rows] if gather else a[:n]
    out = torch.zeros(n, w.shape[1], dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    off = offsets.tolist()
    for e in range(w.shape[0]):
        s = slice(off[e], off[e + 1])
        if off[e + 1] == off[e]:
            continue
        out[s] = src[s].double() @ w[e].double().t()
        bound[s] = _acc_bound(w.shape[2]) * (src[s].double().abs() @ w[e].double().abs().t())
        if b is not None:
            out[s] += b[e].double()
            bound[s] += 2.0**-23 * b[e].double().abs()
    bound += 2.0**-23 * out.abs()
    if gelu:
        out = out * 0.5 * torch.erfc(-out / math.sqrt(2.0))
        bound = 1.13 * bound + 5e-7  # GELU's slope is at most 1.129
    return out, bound


def _check_ffn(cuda_pkg, a, w_in, b_in, w_out, b_out, r, rms=True):
    k = cuda_pkg.kernels
    u = torch.finfo(a.dtype).eps / 2
    off, slot_row = r.offsets, r.slot_row
    h, bh = _ref_gemm(a, w_in, b_in, slot_row, off, True, True)
    got_h = k.gemm_experts(a, w_in, b_in, r, gather=True, gelu=True)
    n = h.shape[0]
    bh = bh + u * (h.abs() + bh) + 1e-7
    assert ((got_h[:n].double() - h).abs() <= bh).all()
    # FFN-out from the kernel's own hidden layer
    y, by = _ref_gemm(got_h, w_out, b_out, slot_row, off, False, False)
    got_y = k.gemm_experts(got_h, w_out, b_out, r, gather=False)
    by = by + u * (y.abs() + by) + 1e-7
    assert ((got_y[:n].double() - y).abs() <= by).all()
    # the whole, from exact values
    y, _ = _ref_gemm(h, w_out, b_out, slot_row, off, False, False)
    ends = off.tolist()
    for e in range(w_out.shape[0]):
        s = slice(ends[e], ends[e + 1])
        by[s] += bh[s] @ w_out[e].double().abs().t()
    out = torch.zeros(a.shape[0], w_out.shape[1], dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    for j in range(r.top_k):
        slot = r.row_slot[:, j].long()
        has = slot >= 0
        out[has] += r.weights[has, j : j + 1].double() * y[slot[has]]
        bound[has] += r.weights[has, j : j + 1].double().abs() * (by[slot[has]] + r.top_k * U32 * y[slot[has]].abs())
    got = k.expert_ffn(a, w_in, b_in, w_out, b_out, r)
    bound = bound + u * (out.abs() + bound) + 1e-7
    err = (got.double() - out).abs()
    assert (err <= bound).all(), float((err / bound).max())
    if rms and out.numel() > 100:
        assert float(err.square().mean().sqrt()) <= 4 * u * float(out.square().mean().sqrt())
    # the same outputs rounded to 16 bits before their sum
    summed = k.expert_combine(got_y, r).double()
    assert ((summed - out).abs() <= bound).all()
    return got


# One token; few tokens per expert (narrow tiles); a tile's edge (16, 32, 256
# tokens of one expert and one more); widths that end inside a tile of 128
# features or 64 columns; many rows of few experts.
@pytest.mark.parametrize("rows,E,k,D,F", [
    (1, 8, 2, 1024, 4096), (1, 1, 1, 8, 8), (5, 64, 4, 64, 128), (33, 4, 2, 200, 328), (16, 1, 1, 64, 64),
    (17, 1, 1, 72, 136), (32, 1, 1, 128, 256), (33, 1, 1, 128, 256), (256, 1, 1, 128, 264), (257, 1, 1, 64, 128),
    (300, 3, 3, 136, 120), (1777, 12, 2, 760, 1912), (4096, 8, 2, 512, 1024), (2000, 300, 2, 64, 72),
    (700, 512, 8, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_expert_ffn(cuda_pkg, rows, E, k, D, F, dtype):
    g = _gen(rows + 3 * E + D)
    r = cuda_pkg.kernels.route_experts(_randn(g, rows, E, std=1.5), k)
    a = _randn(g, rows, D, dtype=dtype)
    b_in, b_out = _randn(g, E, F, std=0.3), _randn(g, E, D, std=0.3)
    _check_ffn(cuda_pkg, a, _weights(g, E, F, D, dtype), b_in, _weights(g, E, D, F, dtype), b_out, r)
    _check_ffn(cuda_pkg, a, _weights(g, E, F, D, dtype), None, _weights(g, E, D, F, dtype), None, r)


@pytest.mark.parametrize("rows", [40, 900])
def test_expert_ffn_skewed_closed_and_repeated(cuda_pkg, rows):
    """All rows on one expert, rows without experts, an expert named twice."""
    g = _gen(rows)
    E, D, F = 16, 128, 192
    w_in, w_out = _weights(g, E, F, D, torch.float16), _weights(g, E, D, F, torch.float16)
    b_in, b_out = _randn(g, E, F), _randn(g, E, D)
    a = _randn(g, rows, D, dtype=torch.float16)
    for first in (0, 15):
        idx = torch.full((rows, 2), first, dtype=torch.int32, device=DEV)  # twice
        idx[::3, 1] = -1
        idx[::7] = -1
        idx[5] = torch.tensor([3, 9], dtype=torch.int32)
        wt = torch.rand(rows, 2, generator=g, device=DEV)
        r = cuda_pkg.kernels.expert_plan(idx, wt, E)
        out = _check_ffn(cuda_pkg, a, w_in, b_in, w_out, b_out, r)
        assert (out[0] == 0).all()
    none = cuda_pkg.kernels.expert_plan(torch.full((rows, 2), -1, dtype=torch.int32, device=DEV), wt, E)
    assert (cuda_pkg.kernels.expert_ffn(a, w_in, b_in, w_out, b_out, none) == 0).all()


def test_expert_ffn_leaves_the_rest(cuda_pkg):
    """Rows past row_count, slots past the last: as they were; NaN in rows nobody routes is not read."""
    k = cuda_pkg.kernels
    g = _gen(3)
    rows, live, E, D, F = 500, 321, 6, 64, 96
    logits = _randn(g, rows, E)
    logits[7] = -math.inf
    count = torch.tensor([live], dtype=torch.int32, device=DEV)
    r = k.route_experts(logits, 2, row_count=count)
    a = _randn(g, rows, D, dtype=torch.float16)
    a[live:] = math.nan
    a[7] = math.nan
    w_in, w_out = _weights(g, E, F, D, torch.float16), _weights(g, E, D, F, torch.float16)
    mark = torch.full((rows, D), 7.0, dtype=torch.float16, device=DEV)
    out = k.expert_ffn(a, w_in, None, w_out, None, r, out=mark)
    assert (out[live:] == 7).all() and (out[7] == 0).all() and not torch.isnan(out).any()
    n = int(r.offsets[-1])
    assert n == 2 * (live - 1)
    h = torch.full((rows * 2, F), 5.0, dtype=torch.float16, device=DEV)
    k.gemm_experts(a, w_in, None, r, gather=True, gelu=True, out=h)
    assert (h[n:] == 5).all() and not torch.isnan(h).any()
    h[n:] = math.nan
    y = torch.full((rows * 2, D), 3.0, dtype=torch.float16, device=DEV)
    k.gemm_experts(h, w_out, None, r, gather=False, out=y)
    assert (y[n:] == 3).all() and not torch.isnan(y).any()
    y[n:] = math.nan
    mark.fill_(2.0)
    summed = k.expert_combine(y, r, out=mark)
    assert not torch.isnan(summed).any() and (summed[live:] == 2).all() and (summed[7] == 0).all()


def test_expert_ffn_past_32_bit_offsets(cuda_pkg):
    """rows * top_k * F above 2^31 elements."""
    k = cuda_pkg.kernels
    g = _gen(4)
    rows, E, D, F = 530_000, 4, 64, 4096
    r = k.route_experts(_randn(g, rows, E), 1)
    a = _randn(g, rows, D, dtype=torch.bfloat16)
    w_in, w_out = _weights(g, E, F, D, torch.bfloat16), _weights(g, E, D, F, torch.bfloat16)
    h = k.gemm_experts(a, w_in, None, r, gather=True, gelu=True)
    assert h.numel() > 2**31
    u = torch.finfo(torch.bfloat16).eps / 2
    for s in (0, 262_144, 524_288, rows - 1):  # 2^31 / F = 524288
        e = int((r.offsets[1:] <= s).sum())
        z = w_in[e].double() @ a[int(r.slot_row[s])].double()
        ref = z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
        bound = 1.13 * _acc_bound(D) * (w_in[e].double().abs() @ a[int(r.slot_row[s])].double().abs()) + 5e-7
        assert ((h[s].double() - ref).abs() <= bound + u * (ref.abs() + bound) + 1e-7).all()
    y = k.gemm_experts(h, w_out, None, r, gather=False)
    s = rows - 1
    e = int((r.offsets[1:] <= s).sum())
    ref = w_out[e].double() @ h[s].double()
    bound = _acc_bound(F) * (w_out[e].double().abs() @ h[s].double().abs())
    assert ((y[s].double() - ref).abs() <= bound + u * (ref.abs() + bound) + 1e-7).all()


# ---- sandwich norm ---------------------------------------------------------------
def _norm64(v, kind, gamma, beta, eps):
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    n = c / torch.sqrt(c.square().mean(1, keepdim=True) + eps)
    y = n * gamma.double()
    amp = n.abs().amax(1, keepdim=True) * gamma.double().abs()
    if beta is not None:
        y = y + beta.double()
        amp = amp + beta.double().abs()
    return y, amp


def _check_sandwich(cuda_pkg, x, branch, pre_g, pre_b=None, post_g=None, post_b=None, kind="layer", gate=None, act="none",
                    per_gate=1, gate_map=None, scale=1.0, eps=1e-5, row_map=None, live=None, routing=None):
    u = torch.finfo(branch.dtype).eps / 2
    count = None if live is None else torch.tensor([live], dtype=torch.int32, device=DEV)
    rows = branch.shape[0] if routing is None else routing.rows
    D = x.shape[1]
    s_out = torch.full((rows, D), 9.0, device=DEV)
    y_out = torch.full((rows, D), 8.0, dtype=branch.dtype, device=DEV)
    s, y = cuda_pkg.kernels.sandwich_norm(
        x, branch, pre_g, pre_b, post_gamma=post_g, post_beta=post_b, kind=kind, gate=gate, gate_act=act,
        rows_per_gate=per_gate, gate_map=gate_map, residual_scale=scale, eps=eps, row_map=row_map, row_count=count,
        routing=routing, sum_out=s_out, out=y_out)
    n = rows if live is None else min(rows, live)
    assert (s[n:] == 9).all() and (y[n:] == 8).all()
    src = torch.arange(n, device=DEV) if row_map is None else row_map[:n].long()
    if routing is None:
        b, amp_b = branch[:n].double(), branch[:n].double().abs()
    else:
        b = torch.zeros(n, D, dtype=torch.float64, device=DEV)
        amp_b = torch.zeros_like(b)
        for j in range(routing.top_k):
            slot = routing.row_slot[:n, j].long()
            part = torch.where(slot[:, None] >= 0, branch.double()[slot.clamp(min=0)], 0.0) * routing.weights[:n, j : j + 1].double()
            b += part
            amp_b += part.abs()
    amp = amp_b * 1.0
    if post_g is not None:
        spread = torch.sqrt((b.var(1, unbiased=False, keepdim=True) if kind == "layer" else b.square().mean(1, keepdim=True)) + eps)
        noise = amp_b.amax(1, keepdim=True) / spread  # of a summed branch, before its norm
        b, amp = _norm64(b, kind, post_g, post_b, eps)
        amp = amp + noise * post_g.double().abs()
    if gate is not None:
        gt = gate.double()
        if act == "sigmoid":
            gt = torch.sigmoid(gt)
        elif act == "tanh":
            gt = torch.tanh(gt)
        if gate.dim() == 2:
            gm = gate_map if gate_map is not None else row_map
            gsrc = torch.arange(n, device=DEV) if gm is None else gm[:n].long()
            gt = gt[gsrc // per_gate]
        b, amp = b * gt, amp * gt.abs()
    ref = x.double()[src] + scale * b
    tol = 128 * U32 * (x.double()[src].abs() + abs(scale) * amp)
    assert ((s[:n].double() - ref).abs() <= tol + 1e-30).all()
    yr, amp = _norm64(s[:n].double(), kind, pre_g, pre_b, eps)  # of the kernel's own sum
    tol = 128 * U32 * amp
    assert ((y[:n].double() - yr).abs() <= tol + u * (yr.abs() + tol) + 1e-7).all()


def _affine(g, D):
    return 1.0 + 0.2 * _randn(g, D), 0.1 * _randn(g, D)


# Every split of a row over threads: one warp (up to 1024 columns), 128 and 512
# threads, each with and without whole groups of 8 columns.
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 1024), (9, 8), (5, 31), (64, 256), (33, 264), (70, 512), (17, 513),
                                    (100, 1000), (1000, 1021), (65, 1032), (40, 2048), (11, 2049), (7, 4096), (5, 4097),
                                    (3, 8191), (3, 8192), (2, 16384), (2, 32768), (4097, 1024)])
@pytest.mark.parametrize("dtype,kind", [(torch.float16, "layer"), (torch.bfloat16, "rms")])
def test_sandwich_norm(cuda_pkg, rows, D, dtype, kind):
    g = _gen(rows + D)
    x, b = _randn(g, rows, D, std=2.0), _randn(g, rows, D, dtype=dtype, std=1.5)
    pg, pb = _affine(g, D)
    qg, qb = _affine(g, D)
    beta = kind == "layer"
    _check_sandwich(cuda_pkg, x, b, pg, pb if beta else None, qg, qb if beta else None, kind)
    _check_sandwich(cuda_pkg, x, b, pg, None, None, None, kind, gate=_randn(g, D), scale=0.5)
    _check_sandwich(cuda_pkg, x, b, pg, pb, qg, None, kind, gate=_randn(g, rows, D, dtype=dtype), act="sigmoid", scale=-2.0)


# Enough rows that they go through shared memory: every split of a row, whole
# and partly filled, aligned and not; in place.
@pytest.mark.parametrize("rows,D", [(700, 1), (700, 8), (1200, 31), (3000, 256), (700, 264), (700, 512), (701, 513),
                                    (700, 1000), (700, 1032), (2000, 2048), (700, 2049), (350, 3000), (400, 4095), (900, 4096)])
@pytest.mark.parametrize("dtype,kind", [(torch.float16, "layer"), (torch.bfloat16, "rms")])
def test_sandwich_norm_many_rows(cuda_pkg, rows, D, dtype, kind):
    g = _gen(rows + D)
    x, b = _randn(g, rows, D, std=2.0), _randn(g, rows, D, dtype=dtype, std=1.5)
    pg, pb = _affine(g, D)
    qg, qb = _affine(g, D)
    _check_sandwich(cuda_pkg, x, b, pg, pb, qg, qb, kind, gate=_randn(g, D), act="sigmoid", scale=0.5, live=rows - 3)
    _check_sandwich(cuda_pkg, x, b, pg, None, None, None, kind, gate=_randn(g, rows, D, dtype=dtype), act="tanh")
    _check_sandwich(cuda_pkg, x, b, pg, pb, qg, None, kind, gate=_randn(g, -(-rows // 64), D), per_gate=64)
    s0, y0 = cuda_pkg.kernels.sandwich_norm(x, b, pg, pb, post_gamma=qg, kind=kind)
    s, y = cuda_pkg.kernels.sandwich_norm(x, b, pg, pb, post_gamma=qg, kind=kind, sum_out=x, out=b)
    assert s is x and y is b and torch.equal(s, s0) and torch.equal(y, y0)


def test_sandwich_norm_of_more_experts_than_fit(cuda_pkg):
    """16 and 32 experts' rows of 4096 columns: one row or none in shared memory."""
    g = _gen(12)
    for k, rows in ((6, 400), (16, 320), (32, 310)):
        r = cuda_pkg.kernels.route_experts(_randn(g, rows, 40), k)
        y = _randn(g, rows * k, 4096, dtype=torch.float16)
        pg, pb = _affine(g, 4096)
        _check_sandwich(cuda_pkg, _randn(g, rows, 4096), y, pg, pb, pg, pb, gate=_randn(g, 4096), routing=r)


def test_sandwich_norm_past_32_bit_offsets(cuda_pkg):
    """rows * D above 2^31 elements."""
    g = _gen(13)
    rows, D = 524_500, 4096
    x = torch.empty(rows, D, device=DEV).normal_(generator=g)
    b = torch.empty(rows, D, device=DEV, dtype=torch.float16).normal_(generator=g)
    pg, pb = _affine(g, D)
    s, y = cuda_pkg.kernels.sandwich_norm(x, b, pg, pb, post_gamma=pg)
    assert s.numel() > 2**31
    for lo in (0, 524_280, rows - 8):  # 2^31 / D = 524288
        part = slice(lo, lo + 8)
        s1, y1 = cuda_pkg.kernels.sandwich_norm(x[part].clone(), b[part].clone(), pg, pb, post_gamma=pg)
        assert (s[part] - s1).abs().max() <= 1e-5 and torch.allclose(y[part].float(), y1.float(), rtol=2**-10, atol=1e-5)


@pytest.mark.parametrize("D", [96, 1021, 2048])
@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
def test_sandwich_norm_gates(cuda_pkg, D, act):
    g = _gen(D)
    rows, S = 333, 50
    x, b = _randn(g, rows, D), _randn(g, rows, D, dtype=torch.float16)
    pg, pb = _affine(g, D)
    qg, qb = _affine(g, D)
    args = (x, b, pg, pb, qg, qb, "layer")
    _check_sandwich(cuda_pkg, *args, gate=4 * _randn(g, D), act=act)
    _check_sandwich(cuda_pkg, *args, gate=4 * _randn(g, 7, D), act=act, per_gate=S)
    _check_sandwich(cuda_pkg, *args, gate=_randn(g, 7, D, dtype=torch.float16), act=act, per_gate=S)
    _check_sandwich(cuda_pkg, *args, gate=_randn(g, rows, D), act=act)
    # packed rows of a padded batch: x at the original rows, a gate per sample
    big = _randn(g, 10 * S, D)
    rm = torch.randperm(10 * S, generator=g, device=DEV)[:rows].sort()[0].int()
    gate = _randn(g, 10, D)
    _check_sandwich(cuda_pkg, big, b, pg, pb, qg, qb, gate=gate, act=act, per_gate=S, row_map=rm, live=300)
    _check_sandwich(cuda_pkg, x, b, pg, pb, qg, qb, gate=gate, act=act, per_gate=S, gate_map=rm)


@pytest.mark.parametrize("rows,E,k,D", [(1, 4, 2, 128), (300, 8, 1, 1024), (300, 16, 3, 2048), (50, 5, 4, 4096), (64, 8, 2, 104)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sandwich_norm_of_experts(cuda_pkg, rows, E, k, D, dtype):
    g = _gen(rows + D)
    logits = _randn(g, rows, E)
    if rows > 1:
        logits[1] = -math.inf
    r = cuda_pkg.kernels.route_experts(logits, k)
    y = _randn(g, rows * k, D, dtype=dtype)
    y[int(r.offsets[-1]) :] = math.nan
    pg, pb = _affine(g, D)
    qg, qb = _affine(g, D)
    x = _randn(g, rows, D)
    _check_sandwich(cuda_pkg, x, y, pg, pb, qg, qb, "layer", gate=_randn(g, rows, D, dtype=dtype), act="tanh", routing=r)
    _check_sandwich(cuda_pkg, x, y, pg, None, None, None, "rms", routing=r, live=rows // 2)


def test_sandwich_norm_flat_and_large_rows(cuda_pkg):
    """A branch of zeros or of one value (variance 0), values near the type's
    largest, NaN rows that stay in their row; the sum in place of x."""
    g = _gen(8)
    x = _randn(g, 64, 768)
    b = _randn(g, 64, 768, dtype=torch.float16)
    b[3] = 0
    b[4] = 5.0
    b[5] = 60000.0 * torch.sign(b[5])
    pg, pb = _affine(g, 768)
    qg, qb = _affine(g, 768)
    _check_sandwich(cuda_pkg, x, b, pg, pb, qg, qb)
    s0, y0 = cuda_pkg.kernels.sandwich_norm(x, b, pg, pb, post_gamma=qg, post_beta=qb)
    b2 = b.clone()
    b2[10, 3] = math.nan
    s, y = cuda_pkg.kernels.sandwich_norm(x, b2, pg, pb, post_gamma=qg, post_beta=qb)
    keep = [i for i in range(64) if i != 10]
    assert torch.isnan(y[10]).all() and torch.equal(y[keep], y0[keep]) and torch.equal(s[keep], s0[keep])
    x2 = x.clone()
    s, y = cuda_pkg.kernels.sandwich_norm(x2, b, pg, pb, post_gamma=qg, post_beta=qb, sum_out=x2)
    assert s.data_ptr() == x2.data_ptr() and torch.equal(s, s0) and torch.equal(y, y0)


def test_sandwich_norm_unaligned(cuda_pkg):
    """Operands off a 16-byte boundary take the one-column path."""
    g = _gen(6)
    D = 264
    flat = _randn(g, 40 * D + 1)
    x = flat[1:].view(40, D)
    b = _randn(g, 40, D, dtype=torch.float16)
    pg, pb = _affine(g, D)
    _check_sandwich(cuda_pkg, x, b, pg, pb)
    _check_sandwich(cuda_pkg, x.clone(), _randn(g, 40 * D + 1, dtype=torch.float16)[1:].view(40, D), pg, pb)


def test_sandwich_norm_reports_bad_rows(cuda_pkg):
    L = cuda_pkg._lib
    g = _gen(1)
    x, b = _randn(g, 20, 64), _randn(g, 20, 64, dtype=torch.float16)
    gamma = torch.ones(64, device=DEV)
    rm = torch.arange(20, dtype=torch.int32, device=DEV)
    for bad in (20, -1):
        m = rm.clone()
        m[4] = bad
        with pytest.raises(L.TJError, match="outside"):
            cuda_pkg.kernels.sandwich_norm(x, b, gamma, row_map=m)
        with pytest.raises(L.TJError, match="outside"):
            cuda_pkg.kernels.sandwich_norm(x, b, gamma, gate=_randn(g, 4, 64), rows_per_gate=5, gate_map=m)
    assert L.device_status(torch.cuda.current_stream().cuda_stream) == [0, 0, 0, 0]


# ---- together --------------------------------------------------------------------
def _block(k, w, x, mask=None):
    """One expert feed-forward block over the packed rows of a padded batch."""
    B, S, D = x.shape
    plan = k.token_plan(mask, B, S, x.device)
    nv, _, _, orig, inv = k.plan_views(plan, B, S)
    a = k.ln_cast_f16(x.view(B * S, D), w["g1"], w["b1"], row_map=orig, row_count=nv)
    logits = torch.nn.functional.linear(a.float(), w["router"])
    r = k.route_experts(logits, 2, scoring="sigmoid", bias=w["balance"], row_count=nv)
    h = k.gemm_experts(a, w["w_in"], w["b_in"], r, gather=True, gelu=True)
    y = k.gemm_experts(h, w["w_out"], w["b_out"], r, gather=False)
    s, n = k.sandwich_norm(x.view(B * S, D), y, w["g3"], w["b3"], post_gamma=w["g2"], post_beta=w["b2"], gate=w["gate"],
                           gate_act="tanh", rows_per_gate=S, residual_scale=0.5, row_map=orig, routing=r)
    return s, n, nv, orig, inv, r, a


def _block_weights(g, B, D, F, E):
    w = {"router": _randn(g, E, D, std=D**-0.5), "balance": _randn(g, E, std=0.02), "gate": _randn(g, B, D),
         "w_in": _weights(g, E, F, D, torch.float16), "b_in": _randn(g, E, F, std=0.1),
         "w_out": _weights(g, E, D, F, torch.float16), "b_out": _randn(g, E, D, std=0.1)}
    for i in "123":
        w["g" + i], w["b" + i] = _affine(g, D)
    return w


def _check_block(w, x, mask, got):
    s, n, nv, orig, inv, r, a = got
    B, S, D = x.shape
    live = int(nv)
    assert live == int(mask.sum())
    rows = orig[:live].long()
    xs = x.view(B * S, D)[rows].double()
    idx, wt = r.experts[:live].long(), r.weights[:live].double()
    out = torch.zeros(live, D, dtype=torch.float64, device=DEV)
    for e in range(w["router"].shape[0]):
        share = torch.where(idx == e, wt, 0.0).sum(1, keepdim=True)
        z = a[:live].double() @ w["w_in"][e].double().t() + w["b_in"][e].double()
        z = z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
        out += share * (z @ w["w_out"][e].double().t() + w["b_out"][e].double())
    p, _ = _norm64(out, "layer", w["g2"], w["b2"], 1e-5)
    ref = xs + 0.5 * torch.tanh(w["gate"].double())[rows // S] * p
    yr, _ = _norm64(ref, "layer", w["g3"], w["b3"], 1e-5)
    # rms as in _check_ffn; the post norm scales error and value alike
    u = torch.finfo(torch.float16).eps / 2
    assert float((s[:live].double() - ref).square().mean().sqrt()) <= 4 * u * float((ref - xs).square().mean().sqrt())
    assert float((n[:live].double() - yr).square().mean().sqrt()) <= 5 * u * float(yr.square().mean().sqrt())


@pytest.mark.parametrize("B,S,D,F,E", [(1, 1, 128, 256, 4), (4, 70, 256, 512, 8), (8, 300, 512, 768, 16)])
def test_block(cuda_pkg, B, S, D, F, E):
    g = _gen(B * S)
    w = _block_weights(g, B, D, F, E)
    x = _randn(g, B, S, D)
    lengths = torch.randint(1, S + 1, (B,), generator=g, device=DEV)
    mask = torch.arange(S, device=DEV)[None] < lengths[:, None]
    _check_block(w, x, mask, _block(cuda_pkg.kernels, w, x, mask))


def test_block_captured_and_on_two_streams(cuda_pkg):
    """A captured block replays on new inputs; two blocks run at once on two
    streams; results equal the eager ones bit for bit."""
    cuda_pkg._lib.set_sync_check(False)
    k = cuda_pkg.kernels
    g = _gen(77)
    B, S, D, F, E = 3, 90, 256, 512, 8
    w = _block_weights(g, B, D, F, E)
    xs = [_randn(g, B, S, D) for _ in range(3)]
    masks = [torch.rand(B, S, generator=g, device=DEV) < p for p in (0.9, 0.2, 0.6)]

    def outputs(got):
        live = int(got[2])
        return got[0][:live].clone(), got[1][:live].clone(), got[5].experts.clone()

    want = [outputs(_block(k, w, x, m)) for x, m in zip(xs, masks)]
    sx, sm = xs[0].clone(), masks[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(k, w, sx, sm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _block(k, w, sx, sm)
    for i in (1, 2, 0):
        sx.copy_(xs[i])
        sm.copy_(masks[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outputs(got), want[i]):
            assert torch.equal(a, b)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for rep in range(5):
        for st, i in zip(streams, (1, 2)):
            with torch.cuda.stream(st):
                results.append((i, _block(k, w, xs[i], masks[i])))
    torch.cuda.synchronize()
    for i, got in results:
        for a, b in zip(outputs(got), want[i]):
            assert torch.equal(a, b)
    assert cuda_pkg._lib.device_status(torch.cuda.current_stream().cuda_stream) == [0, 0, 0, 0]


# ---- given up on -------------------------------------------------------------------
# Products of few rows (TMA row gathers) and of many (CTA pairs after the permuted
# copy), with more K steps than stages.
def _products(k, g, rows, E=4, D=1024, F=768):
    r = k.route_experts(_randn(g, rows, E), 2)
    a = _randn(g, rows, D, dtype=torch.float16)
    w_in, w_out = _weights(g, E, F, D, torch.float16), _weights(g, E, D, F, torch.float16)
    h = torch.empty(rows * 2, F, dtype=torch.float16, device=DEV)

    def run(fill=None):
        if fill is not None:
            h.fill_(fill)
        k.gemm_experts(a, w_in, None, r, gather=True, gelu=True, out=h)
        y = k.gemm_experts(h, w_out, None, r, gather=False)
        return h, y, k.expert_ffn(a, w_in, None, w_out, None, r)

    return run


@pytest.mark.parametrize("rows", [20, 1500])
def test_products_after_a_recorded_error(cuda_pkg, rows):
    """Until the status is read the products load and write nothing; then they are as before."""
    L, k = cuda_pkg._lib, cuda_pkg.kernels
    run = _products(k, _gen(rows), rows)
    want = [t.clone() for t in run()]
    L.set_sync_check(False)
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(5):
        k.expert_plan(torch.full((rows, 2), 9, dtype=torch.int32, device=DEV), torch.ones(rows, 2, device=DEV), 8)
        h, _, _ = run(fill=7.0)
        with pytest.raises(L.TJError, match="outside"):
            L.device_status(stream)
        assert (h == 7).all()
        for got, ref in zip(run(), want):
            assert torch.equal(got, ref)
        assert L.device_status(stream) == [0, 0, 0, 0]


@pytest.mark.parametrize("rows", [20, 1500])
def test_products_whose_waits_run_out(cuda_pkg, rows):
    """A wait limit of 1 ns: producers stop at different steps, everything sent
    lands, and the next products are as before."""
    L, k = cuda_pkg._lib, cuda_pkg.kernels
    lib = L.load()
    run = _products(k, _gen(rows), rows)
    want = [t.clone() for t in run()]
    L.set_sync_check(False)
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(20):
        L.check(lib.tj_debug_set_wait_limit_ns(1), "debug_set_wait_limit_ns")
        try:
            run()
            with pytest.raises(L.TJError, match="time limit"):
                L.device_status(stream)
        finally:
            L.check(lib.tj_debug_set_wait_limit_ns(0), "debug_set_wait_limit_ns")
        for got, ref in zip(run(), want):
            assert torch.equal(got, ref)
        assert L.device_status(stream) == [0, 0, 0, 0]


# ---- routing: rows of many terms, biases far apart, scores that saturate ---------------
def _peaked(rows, E):
    """Softmax rows whose denominator, summed one after the other in fp32, rounds up at every term."""
    logits = torch.full((rows, E), math.log(1.01 * 2.0**-24), device=DEV)
    logits[:, 0] = 0.0
    return logits


# As many terms to a lane as there are (rows many, so few lanes to each): top_k up to
# 16 and above (half the threads), one chunk of rows and many.
@pytest.mark.parametrize("rows,E,k", [(19092, 384, 17), (15000, 512, 24), (30000, 88, 17), (14000, 512, 8), (60, 512, 32)])
def test_route_biased_softmax_of_many_terms(cuda_pkg, rows, E, k):
    logits = _peaked(rows, E)
    p = torch.softmax(logits[0].double(), 0)
    bias = -1.0 - 0.01 * torch.arange(E, device=DEV)
    bias[0] = 0.0
    for below in (3e-7, -3e-7):  # how far expert 1 lies below expert 0
        bias[1] = float(p[0] - p[1] - below)
        r = _check_route(cuda_pkg, logits, k, bias=bias)
        assert int(r.experts[0, 0]) == (0 if below > 0 else 1)


# Tolerance of _check_route: 32 * 2^-24.  The denominator is summed in blocks of 16
# in four parts (5 roundings), at most 13 blocks, and over the lanes (5); expf within
# 2 ulp (4 * 2^-24), the exponents' differences are exact here, two more roundings.
@pytest.mark.parametrize("rows,E,k", [(19092, 384, 17), (15000, 512, 32), (14000, 512, 8), (30000, 88, 20), (60, 512, 32)])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_weights_of_many_terms(cuda_pkg, rows, E, k, renorm):
    _check_route(cuda_pkg, _peaked(rows, E), k, renorm=renorm)
    flat = torch.zeros(rows, E, device=DEV)
    flat[:, 1] = 1.0
    _check_route(cuda_pkg, flat, k, renorm=renorm)
    _check_route(cuda_pkg, _peaked(rows, E), k, "sigmoid", renorm=renorm)


@pytest.mark.parametrize("rows,E,k", [(3000, 100, 17), (15000, 512, 24), (20000, 40, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_more_than_16_of_many_rows(cuda_pkg, rows, E, k, dtype):
    g = _gen(rows + k)
    logits = _randn(g, rows, E, std=1.5).to(dtype)
    bias = _randn(g, E, std=0.02)
    for scoring in ("softmax", "sigmoid"):
        _check_route(cuda_pkg, logits, k, scoring)
        _check_route(cuda_pkg, logits, k, scoring, bias=bias)
        _check_route(cuda_pkg, logits, k, scoring, bias=bias, groups=4, top_groups=4, group_top=2, renorm=False)


@pytest.mark.parametrize("rows,E,k", [(1, 8, 3), (300, 40, 6), (16000, 96, 8), (5000, 200, 17)])
def test_route_scores_that_saturate(cuda_pkg, rows, E, k):
    """Scores whose 64-bit values are equal: the greater logit is the greater score,
    with a bias of zeros as without a bias, and equal logits go by index."""
    g = _gen(rows + E)
    zeros = torch.zeros(E, device=DEV)
    near = torch.randint(40, 60, (rows, E), generator=g, device=DEV).float()  # sigmoid 1 - 4e-18 and nearer to 1
    far = torch.randint(-990, -960, (rows, E), generator=g, device=DEV).float()  # exp 0 beside a logit of 0
    far[:, E - 1] = 0.0
    for logits, scoring in ((near, "sigmoid"), (far, "softmax"), (far, "sigmoid")):
        want = cuda_pkg.kernels.route_experts(logits, k, scoring=scoring)
        order = np.argsort(-logits.cpu().numpy(), axis=1, kind="stable")[:, :k]
        assert np.array_equal(want.experts.cpu().numpy(), order)
        got = cuda_pkg.kernels.route_experts(logits, k, scoring=scoring, bias=zeros)
        assert torch.equal(got.experts, want.experts)
        got = cuda_pkg.kernels.route_experts(logits, k, scoring=scoring, bias=zeros + 0.25)
        assert torch.equal(got.experts, want.experts)
    # a bias decides before a logit does; infinite ones are equal, in index order
    bias = zeros.clone()
    bias[1::2] = 1e-6
    got = cuda_pkg.kernels.route_experts(near, k, scoring="sigmoid", bias=bias).experts.cpu().numpy()
    odd = np.where(np.arange(E)[None] % 2 == 1, near.cpu().numpy(), near.cpu().numpy() - 100.0)
    assert np.array_equal(got, np.argsort(-odd, axis=1, kind="stable")[:, :k])
    bias[2:5] = math.inf
    got = cuda_pkg.kernels.route_experts(near, 3, scoring="sigmoid", bias=bias).experts
    assert (got == torch.tensor([2, 3, 4], device=DEV)).all()


def _fastest(fn, n=10):
    """Least time of n calls on the GPU, in us."""
    times = []
    for i in range(n + 2):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        fn()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end) * 1e3)
    return min(times[2:])


@pytest.mark.parametrize("groups", [1, 8])
def test_route_of_an_expert_disabled_by_its_bias(cuda_pkg, groups):
    """A bias of -1e9 (or the type's lowest) orders like -inf, and costs no more:
    only values that lie near each other are decided again in 64 bits."""
    cuda_pkg._lib.set_sync_check(False)
    k = cuda_pkg.kernels
    g = _gen(31)
    logits = _randn(g, 60000, 64, std=1.5)
    kw = dict(scoring="sigmoid", num_groups=groups, top_groups=min(groups, 3), group_score_top=2)
    names = dict(groups=groups, top_groups=min(groups, 3), group_top=2)
    times = []
    for low in (-math.inf, -1e9, torch.finfo(torch.float32).min):
        bias = _randn(_gen(32), 64, std=0.05)
        bias[[3, 40, 41, 42, 43, 44, 45, 46]] = low  # of one group, all but one
        r = _check_route(cuda_pkg, logits, 6, "sigmoid", bias=bias, **names)
        if low == -math.inf:
            want = r.experts
        assert torch.equal(r.experts, want)
        times.append(_fastest(lambda: k.route_experts(logits, 6, bias=bias, **kw)))
    assert max(times) < 1.5 * times[0], times
    # more choices than experts left: the disabled ones follow, by logit
    few = _randn(g, 500, 16)
    bias = torch.full((16,), torch.finfo(torch.float32).min, device=DEV)
    bias[5] = bias[9] = 0.01
    for gr in (1, 4):
        got = k.route_experts(few, 8, scoring="sigmoid", bias=bias, num_groups=gr, top_groups=gr, group_score_top=2).experts
        first = few.clone()
        first[:, [5, 9]] += 1e4
        assert torch.equal(got.long(), first.sort(stable=True, dim=1, descending=True)[1][:, :8])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("groups", [1, 8])
def test_route_of_equal_values(cuda_pkg, dtype, groups):
    """16-bit logits under a bias of zeros, of one value and of a few steps: the
    order is that of the logits inside each bias, at the cost of any other."""
    cuda_pkg._lib.set_sync_check(False)
    k = cuda_pkg.kernels
    g = _gen(33)
    logits = _randn(g, 30000, 256, std=1.5).to(dtype)
    names = dict(groups=groups, top_groups=min(groups, 4), group_top=1)
    kw = dict(scoring="sigmoid", num_groups=groups, top_groups=min(groups, 4), group_score_top=1)
    spread = _randn(g, 256, std=0.05)
    any_other = _fastest(lambda: k.route_experts(logits, 8, bias=spread, **kw))
    for bias in (torch.zeros(256, device=DEV), torch.full((256,), 0.3, device=DEV),
                 torch.randint(-3, 4, (256,), generator=g, device=DEV) * 0.001, spread):
        for scoring in ("sigmoid", "softmax"):
            _check_route(cuda_pkg, logits, 8, scoring, bias=bias, **names)
        assert _fastest(lambda: k.route_experts(logits, 8, bias=bias, **kw)) < 1.5 * any_other
    _check_route(cuda_pkg, logits, 8, "sigmoid", bias=spread, **(names | dict(group_top=2)))
    _check_route(cuda_pkg, logits, 8, "softmax", **(names | dict(group_top=2)))


@pytest.mark.parametrize("rows", [1, 20, 64, 65, 1500])
def test_expert_ffn_captured_and_on_two_streams(cuda_pkg, rows):
    """Router and FFN with nothing between their kernels: back to back (FFN-out loads
    weights before FFN-in has ended, the next call reuses the workspace's memory),
    captured and replayed on new inputs, and two at once; bit equal to one alone."""
    cuda_pkg._lib.set_sync_check(False)
    k = cuda_pkg.kernels
    g = _gen(rows)
    E, D, F = 4, 512, 1024  # 32 slots per expert at 64 rows
    w_in, w_out = _weights(g, E, F, D, torch.float16), _weights(g, E, D, F, torch.float16)
    b_in, b_out = _randn(g, E, F), _randn(g, E, D)
    inputs = [(_randn(g, rows, E), _randn(g, rows, D, dtype=torch.float16)) for _ in range(4)]

    def run(logits, a):
        r = k.route_experts(logits, 2)
        return k.expert_ffn(a, w_in, b_in, w_out, b_out, r)

    want = []
    for logits, a in inputs:
        want.append(run(logits, a))
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    outs = [(i, run(*inputs[i])) for _ in range(10) for i in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in outs)
    graphs = []
    for n in (1, 2):  # two graphs, of one call and of two
        logits, a = inputs[0][0].clone(), inputs[0][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [run(logits, a) for _ in range(n)]
        graphs.append((graph, logits, a, got))
    for i in (1, 2, 3, 0):
        for graph, logits, a, _ in graphs:
            logits.copy_(inputs[i][0])
            a.copy_(inputs[i][1])
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[i]) for *_, got in graphs for out in got)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for s, i in zip(streams, (1, 2)):
            with torch.cuda.stream(s):
                outs.append((i, run(*inputs[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in outs)
    assert cuda_pkg._lib.device_status(torch.cuda.current_stream().cuda_stream) == [0, 0, 0, 0]


def test_expert_ffn_in_place(cuda_pkg):
    k = cuda_pkg.kernels
    for rows in (7, 400):
        g = _gen(rows)
        a = _randn(g, rows, 64, dtype=torch.bfloat16)
        w_in, w_out = _weights(g, 4, 128, 64, torch.bfloat16), _weights(g, 4, 64, 128, torch.bfloat16)
        r = k.route_experts(_randn(g, rows, 4), 2)
        want = k.expert_ffn(a, w_in, None, w_out, None, r)
        assert k.expert_ffn(a, w_in, None, w_out, None, r, out=a) is a and torch.equal(a, want)


@pytest.mark.parametrize("rows,D", [(700, 64), (2500, 1021), (900, 4096)])
def test_sandwich_norm_skips_bad_rows_of_many(cuda_pkg, rows, D):
    """Map entries, gate rows and slots outside their buffers, spread over teams and
    stages of the shared-memory path: recorded, those rows left as they were (a
    bad slot's share left out), all others as without them."""
    L, k = cuda_pkg._lib, cuda_pkg.kernels
    L.set_sync_check(False)
    stream = torch.cuda.current_stream().cuda_stream
    g = _gen(rows)
    x, b = _randn(g, rows, D), _randn(g, rows, D, dtype=torch.float16)
    pg, pb = _affine(g, D)
    gate = _randn(g, 8, D)
    per = -(-rows // 8)
    rm = torch.randperm(rows, generator=g, device=DEV).int()
    bad = torch.arange(rows, device=DEV) % 7 == 3
    bad[-1] = bad[0] = True
    broken = torch.where(bad, torch.where(rm % 2 == 0, rows + 5, -4), rm).int()

    def run(row_map=None, gate_map=None):
        s, y = torch.full((rows, D), 9.0, device=DEV), torch.full((rows, D), 8.0, dtype=torch.float16, device=DEV)
        return k.sandwich_norm(x, b, pg, pb, post_gamma=pg, gate=gate, rows_per_gate=per, row_map=row_map,
                               gate_map=gate_map, sum_out=s, out=y)

    for good, kw in ((run(rm), dict(row_map=broken)), (run(None, rm), dict(gate_map=torch.where(bad, 8 * per, rm).int()))):
        assert L.device_status(stream) == [0, 0, 0, 0]
        s, y = run(**kw)
        with pytest.raises(L.TJError, match="outside"):
            L.device_status(stream)
        assert (s[bad] == 9).all() and (y[bad] == 8).all()
        assert torch.equal(s[~bad], good[0][~bad]) and torch.equal(y[~bad], good[1][~bad])
    r = k.route_experts(_randn(g, rows, 5), 2)
    y2 = _randn(g, rows * 2, D, dtype=torch.float16)
    r.row_slot[bad, 1] = 2 * rows  # one past the branch
    got = k.sandwich_norm(x, y2, pg, pb, post_gamma=pg, routing=r)
    with pytest.raises(L.TJError, match="outside"):
        L.device_status(stream)
    r.row_slot[bad, 1] = -1
    want = k.sandwich_norm(x, y2, pg, pb, post_gamma=pg, routing=r)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert L.device_status(stream) == [0, 0, 0, 0]


def test_route_groups_of_saturated_scores(cuda_pkg):
    """Strengths of one value that are equal in 64 bits follow its logit, with any
    bias as without one; equal logits go by group."""
    g = _gen(42)
    rows, G, per = 3000, 8, 6
    logits = torch.randint(40, 60, (rows, G * per), generator=g, device=DEV).float()
    kw = dict(scoring="sigmoid", num_groups=G, top_groups=3, group_score_top=1)
    want = cuda_pkg.kernels.route_experts(logits, 8, **kw).experts
    for odd in (0.0, -0.5):  # of one expert, which is then out of it
        bias = torch.zeros(G * per, device=DEV)
        bias[7] = odd
        if odd:
            logits[:, 7] = -50.0
            want = cuda_pkg.kernels.route_experts(logits, 8, **kw).experts
        assert torch.equal(cuda_pkg.kernels.route_experts(logits, 8, bias=bias, **kw).experts, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 3000])
def test_route_far_sigmoids_keep_their_share(cuda_pkg, dtype, rows):
    """Scores down to the subnormals beside small ones, renormalised: as _check_route, and
    where a score is subnormal (steps of 2^-149, two of them in it) that over the sum."""
    g = _gen(rows)
    logits = (torch.randint(-200, -20, (rows, 12), generator=g, device=DEV) * 0.5).to(dtype)
    logits[:, 3] = (torch.randint(-136, -120, (rows,), generator=g, device=DEV) * 0.5).to(dtype)
    for k in (2, 5, 12):
        for renorm in (True, False):
            r = cuda_pkg.kernels.route_experts(logits, k, scoring="sigmoid", renormalize=renorm)
            idx, w = _ref_route(logits, k, "sigmoid", renorm=renorm)
            assert np.array_equal(r.experts.cpu().numpy(), idx)
            total = 1.0 / (1.0 + np.exp(-np.take_along_axis(logits.double().cpu().numpy(), idx, 1)))
            # sums below 1e-30 are of exponentials beside the greatest
            step = np.where(total.sum(1) >= 1e-30, 2.0**-147 / total.sum(1), 2.0**-147)[:, None] if renorm else 2.0**-147
            err = np.abs(r.weights.double().cpu().numpy() - w)
            assert (err <= 32 * U32 * w + step).all(), (err / w).max()
