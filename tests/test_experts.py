"""The mixture-of-experts operators: router, grouped W8A8 product, 4-bit
matrix-vector product, weighted combine, and the feed-forward made of them.

GPU: each against a plain implementation in 64 bits (integers and the W8A8
rounding sequence exactly).  Tolerances are sums of what the operators' own
roundings may do, stated where they are used; half a step of a dtype is
``torch.finfo(dt).eps / 2`` of the value.  CPU: refusals and fake shapes.
"""
import math

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from conftest import cuda_ok

gpu = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]
TDT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = 2.0 ** -24  # half a float32 step


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, generator=gen(seed))


# ---------------------------------------------------------------------------
# plain implementations
# ---------------------------------------------------------------------------


def route_ref(logits, k, scoring, renorm):
    """Token by token in float64; ids, weights, offsets, rows, pos."""
    v = logits.double().numpy()
    T, E = v.shape
    ids, w, pos = np.full((T, k), -1), np.zeros((T, k)), np.full((T, k), -1)
    for t in range(T):
        can = [e for e in range(E) if v[t, e] > -math.inf]
        best = sorted(can, key=lambda e: (-v[t, e], e))[:k]
        ids[t, :len(best)] = best
        if not best:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            if scoring == "softmax":
                ex = np.exp(v[t] - v[t, best[0]])
                g = ex[best] / ex.sum()
                if renorm:
                    g = ex[best] / ex[best].sum() if not np.isnan(v[t]).any() else g
            elif renorm:  # through the logarithm: sigmoids far below zero vanish in any format
                l = np.array([min(v[t, e], 0.0) - math.log1p(math.exp(-abs(v[t, e]))) for e in best])
                g = np.exp(l - l.max())
                g = g / g.sum()
            else:
                g = 1 / (1 + np.exp(-v[t, best]))
        w[t, :len(best)] = g
    offsets, rows = [0], []
    for e in range(E):
        for t in range(T):
            for j in range(k):
                if ids[t, j] == e:
                    pos[t, j] = len(rows)
                    rows.append(t)
        offsets.append(len(rows))
    rows += [-1] * (T * k - len(rows))
    return ids, w, np.array(offsets), np.array(rows), pos


def spans(offsets, R):
    """The rows of each expert as the operators read any offsets."""
    out, at = [], min(max(int(offsets[0]), 0), R)
    for o in offsets[1:]:
        end = min(max(at, int(o)), R)
        out.append((at, end))
        at = end
    return out


def grouped_ref(a, xs, w, ws, offsets, a_rows, bias, dt):
    R = a.shape[0] if a_rows is None else len(a_rows)
    src = torch.arange(R) if a_rows is None else a_rows.long()
    ok = (src >= 0) & (src < a.shape[0])
    src = src.clamp(0, a.shape[0] - 1)
    x = torch.where(ok[:, None], a[src].double(), torch.zeros(()).double())
    s = torch.where(ok, xs.reshape(-1)[src], torch.zeros(()))
    y = torch.zeros(R, w.shape[1], dtype=dt)
    for e, (b, t) in enumerate(spans(offsets, R)):
        acc = (x[b:t] @ w[e].double().T).to(torch.int64)  # exact: below 2^53
        f = acc.float() * s[b:t, None] * ws[e][None]
        f = f.to(dt)
        y[b:t] = f if bias is None else (f.float() + bias[e].float()).to(dt)
    return y


def unpack(p):
    c = p.int() & 255
    return torch.stack(((c % 16 + 8) % 16 - 8, (c // 16 + 8) % 16 - 8), -1).flatten(-2).double()


def matvec_ref(x, p, s, bias, offsets, x_rows):
    """(y, sum of the magnitudes) in float64."""
    q = unpack(p)
    K = q.shape[-1]
    s = s.double()
    if s.dim() == p.dim() and s.shape[-1] != 1:
        w = q * s.repeat_interleave(128, -1)
    else:
        w = q * s.reshape(*p.shape[:-1], 1)
    src = torch.arange(x.shape[0]) if x_rows is None else x_rows.long()
    ok = (src >= 0) & (src < x.shape[0])
    X = torch.where(ok[:, None], x.double()[src.clamp(0, x.shape[0] - 1)], torch.zeros(()).double())
    if offsets is None:
        w, bias, parts = w[None], None if bias is None else bias[None], [(0, len(src))]
    else:
        parts = spans(offsets, len(src))
    y = torch.zeros(len(src), w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for e, (b, t) in enumerate(parts):
        y[b:t] = X[b:t] @ w[e].T
        mag[b:t] = X[b:t].abs() @ w[e].abs().T
        if bias is not None:
            y[b:t] += bias[e].double()
            mag[b:t] += bias[e].double().abs()
    return y, mag


def assert_matvec(got, y, mag, K):
    """A float32 chain adds at most K/16 matrix-instruction steps, the
    groups' multiply-adds and the parts' sums, each within 2^-22 of the
    magnitude (16 products aligned and cut off at 24 bits or more); then
    half a step of the result's dtype."""
    dt = got.dtype
    tol = (K / 16 + K / 128 + 40) * 2.0 ** -22 * mag + torch.finfo(dt).eps / 2 * 1.001 * y.abs() + \
        torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ((got.cpu().double() - y).abs() > tol).sum().item()
    assert bad == 0, f"{bad} of {y.numel()} values off"


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------


def check_route(pkg, logits, k, scoring, renorm, fn=None):
    got = (fn or pkg.ops.route_experts)(logits.cuda(), k, scoring, renorm)
    ids, w, offsets, rows, pos = [t.cpu() for t in got]
    rid, rw, roff, rrows, rpos = route_ref(logits, k, scoring, renorm)
    np.testing.assert_array_equal(ids.numpy(), rid)
    np.testing.assert_array_equal(offsets.numpy(), roff)
    np.testing.assert_array_equal(rows.numpy(), rrows)
    np.testing.assert_array_equal(pos.numpy(), rpos)
    # the exponential's argument is rounded once or twice (half a step of at
    # most the logits' spread, as a relative error of the result), the
    # exponential is within 2 steps, a sum of 21 adds and a division follow
    v = logits.double()
    v = v[torch.isfinite(v)]
    spread = float(v.max() - v.min()) + float(v.abs().max()) if v.numel() else 0.0
    tol = (2 * min(spread, 110.0) + 40) * U
    # below float32's normal range one step is absolute
    np.testing.assert_allclose(w.numpy(), rw, rtol=tol, atol=2.0 ** -148)
    assert w.dtype == torch.float32 and ids.dtype == offsets.dtype == rows.dtype == pos.dtype == torch.int32


@on_gpu
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 6), (3, 5, 5), (64, 32, 4), (65, 33, 2), (130, 60, 4),
                                   (257, 128, 8), (1000, 257, 3), (700, 512, 32), (5000, 16, 2), (19001, 7, 1)])
@pytest.mark.parametrize("scoring,renorm,dt", [("softmax", True, "bf16"), ("softmax", False, "f32"),
                                               ("sigmoid", True, "f32"), ("sigmoid", False, "f16")])
def test_route(pkg, T, E, k, scoring, renorm, dt):
    if T > 4000 and (scoring, renorm) not in (("softmax", True), ("sigmoid", False)):
        pytest.skip("long sorts once a scoring")
    check_route(pkg, (randn(T + E, T, E) * 2).to(TDT[dt]), k, scoring, renorm)


@on_gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_masks_ties_and_extremes(pkg, scoring, renorm):
    x = randn(1, 90, 40)
    x[:, 7] = -math.inf            # an expert switched off
    x[5] = -math.inf               # a token without experts
    x[6, 3:] = -math.inf           # fewer experts than slots
    x[7] = 0.0                     # all tie
    x[8, ::2], x[8, 1::2] = 0.0, -0.0
    x[9] = torch.finfo(torch.float32).min
    x[10] = -120.0                 # sigmoids below float32's range
    x[11, 20] = 80.0
    x[12] = 3.0e38
    check_route(pkg, x, 5, scoring, renorm)


@on_gpu
@pytest.mark.parametrize("renorm", [True, False])
def test_route_nan_and_inf(pkg, renorm):
    x = randn(2, 70, 12)
    x[3, 4] = math.nan
    x[4] = math.nan
    x[5, 2] = math.inf
    ids, w, offsets, rows, pos = [t.cpu() for t in pkg.ops.route_experts(x.cuda(), 3, "softmax", renorm)]
    rid, rw, roff, rrows, rpos = route_ref(x, 3, "softmax", renorm)
    for a, b in ((ids, rid), (offsets, roff), (rows, rrows), (pos, rpos)):
        np.testing.assert_array_equal(a.numpy(), b)
    assert 4 not in ids[3] and w[3].isnan().all()
    assert (ids[4] == -1).all() and (w[4] == 0).all()
    assert ids[5, 0] == 2 and w[5].isnan().all()
    good = [t for t in range(70) if t not in (3, 4, 5)]
    assert torch.isfinite(w[good]).all()
    s = pkg.ops.route_experts(x.cuda(), 3, "sigmoid", False)[1].cpu()
    assert torch.isfinite(s).all() and s[5, 0] == 1.0


@on_gpu
def test_route_strided_and_empty(pkg):
    wide = randn(3, 50, 100)
    x = wide.cuda()[:, 20:53]
    assert not x.is_contiguous()
    for a, b in zip(pkg.ops.route_experts(x, 4), pkg.ops.route_experts(x.contiguous(), 4)):
        assert torch.equal(a, b)
    for a, b in zip(pkg.ops.route_experts(x.T.contiguous().T, 4), pkg.ops.route_experts(x.contiguous(), 4)):
        assert torch.equal(a, b)
    ids, w, offsets, rows, pos = pkg.ops.route_experts(x[:0], 4)
    assert ids.shape == w.shape == pos.shape == (0, 4) and rows.shape == (0,)
    assert offsets.tolist() == [0] * 34


# ---------------------------------------------------------------------------
# grouped W8A8 product
# ---------------------------------------------------------------------------


def grouped_inputs(seed, Ra, E, Nn, K, dt, bias, extreme=False):
    g = gen(seed)
    lo, hi = (-128, 128) if extreme else (-127, 128)
    a = torch.randint(lo, hi, (Ra, K), generator=g).to(torch.int8)
    w = torch.randint(lo, hi, (E, Nn, K), generator=g).to(torch.int8)
    if extreme:
        a[:], w[:] = -128, -128
    xs = torch.rand(Ra, 1, generator=g) * 1e-2 + 1e-4
    ws = torch.rand(E, Nn, generator=g) * 1e-3 + 1e-5
    b = (torch.randn(E, Nn, generator=g)).to(TDT[dt]) if bias else None
    return a, xs, w, ws, b


def run_grouped(pkg, a, xs, w, ws, offsets, a_rows, b, dt):
    c = lambda t: None if t is None else t.cuda()
    return pkg.ops.gemm_w8a8_grouped(c(a), c(xs), c(w), c(ws), torch.tensor(offsets, dtype=torch.int32).cuda(),
                                     c(a_rows), c(b), TDT[dt])


def cum(counts):
    return [0] + list(np.cumsum(counts))


GROUPED = [
    # counts, N, K, dtype, bias
    ([1], 1, 16, "bf16", False),
    ([3], 256, 128, "f32", True),
    ([0, 5, 0], 40, 48, "f16", True),
    ([1, 1, 1, 1], 512, 1024, "bf16", False),
    ([16, 17, 31, 32, 33], 130, 144, "bf16", True),
    ([255, 256, 257, 0, 1], 256, 256, "bf16", False),
    ([100, 300, 513], 257, 400, "f16", True),
    ([64] * 12, 96, 64, "f32", False),
    ([1200, 7], 640, 1040, "bf16", True),
    ([0] * 30 + [2] + [0] * 33, 333, 512, "bf16", False),
]


@on_gpu
@pytest.mark.parametrize("counts,Nn,K,dt,bias", GROUPED)
@pytest.mark.parametrize("gather", [False, True])
def test_grouped(pkg, counts, Nn, K, dt, bias, gather):
    R, E = sum(counts), len(counts)
    Ra = max(1, R // 2) if gather else R
    a, xs, w, ws, b = grouped_inputs(R + Nn, Ra, E, Nn, K, dt, bias)
    rows = torch.randint(0, Ra, (R,), generator=gen(5)).to(torch.int32) if gather else None
    got = run_grouped(pkg, a, xs, w, ws, cum(counts), rows, b, dt)
    want = grouped_ref(a, xs, w, ws, cum(counts), rows, b, TDT[dt])
    assert torch.equal(got.cpu(), want)
    assert pkg.ops.device_error() == 0


@on_gpu
def test_grouped_equals_the_dense_gemm(pkg):
    counts = [300, 0, 129, 512]
    a, xs, w, ws, b = grouped_inputs(11, sum(counts), 4, 384, 512, "bf16", True)
    got = run_grouped(pkg, a, xs, w, ws, cum(counts), None, b, "bf16")
    for e, (s, t) in enumerate(spans(cum(counts), sum(counts))):
        if t > s:
            y = pkg.ops.gemm_w8a8(a[s:t].cuda(), xs[s:t].cuda(), w[e].cuda(), ws[e].cuda(), b[e].cuda())
            assert torch.equal(got[s:t], y)


@on_gpu
@pytest.mark.parametrize("offsets", [[0, 4, 9, 9], [3, 10, 12, 20], [0, 0, 0, 0], [-7, 5, 2, 90], [0, 12, 3, 8],
                                     [40, 50, 60, 70], [2 ** 31 - 1, -2 ** 31, 0, 5]])
def test_grouped_any_offsets_are_safe(pkg, offsets):
    a, xs, w, ws, b = grouped_inputs(12, 24, 3, 72, 160, "bf16", True)
    got = run_grouped(pkg, a, xs, w, ws, offsets, None, b, "bf16")
    assert torch.equal(got.cpu(), grouped_ref(a, xs, w, ws, offsets, None, b, torch.bfloat16))


@on_gpu
def test_grouped_gather_outside_is_zero(pkg):
    a, xs, w, ws, b = grouped_inputs(13, 10, 2, 64, 128, "f32", True)
    rows = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, -2 ** 31, 3, 3], dtype=torch.int32)
    got = run_grouped(pkg, a, xs, w, ws, [0, 5, 8], rows, b, "f32")
    assert torch.equal(got.cpu(), grouped_ref(a, xs, w, ws, [0, 5, 8], rows, b, torch.float32))


@on_gpu
def test_indices_beyond_int32_stay_outside(pkg):
    a, xs, w, ws, _ = grouped_inputs(17, 4, 1, 32, 64, "f32", False)
    rows = torch.tensor([2 ** 32 + 1, -2 ** 32 + 1, 1], dtype=torch.int64).cuda()
    off = torch.tensor([0, 2 ** 33], dtype=torch.int64).cuda()
    y = pkg.ops.gemm_w8a8_grouped(a.cuda(), xs.cuda(), w.cuda(), ws.cuda(), off, rows, None, torch.float32)
    assert (y[:2] == 0).all() and (y[2] != 0).any()
    c = pkg.ops.combine_experts(y, torch.ones(1, 2, device="cuda"), torch.tensor([[2, 2 ** 32]]).cuda())
    assert torch.equal(c[0], y[2])


@on_gpu
def test_grouped_extreme_codes_and_depth(pkg):
    # 128 * 128 * 131056 = 2^31 - 2^18: the largest sum the depth limit lets through
    a, xs, w, ws, _ = grouped_inputs(14, 3, 2, 33, 131056, "f32", False, extreme=True)
    got = run_grouped(pkg, a, xs, w, ws, [0, 1, 3], None, None, "f32")
    assert torch.equal(got.cpu(), grouped_ref(a, xs, w, ws, [0, 1, 3], None, None, torch.float32))


@on_gpu
def test_grouped_odd_depth_and_layouts(pkg):
    """K off 16 is padded; strided operands, 64-bit indices and an unaligned
    base are taken as the other GEMMs take them."""
    counts = [5, 20, 9]
    a, xs, w, ws, b = grouped_inputs(15, 34, 3, 50, 203, "bf16", True)
    want = grouped_ref(a, xs, w, ws, cum(counts), None, b, torch.bfloat16)
    wide = torch.zeros(34, 300, dtype=torch.int8)
    wide[:, 7:210] = a
    off = torch.tensor(cum(counts), dtype=torch.int64).cuda()
    got = pkg.ops.gemm_w8a8_grouped(wide.cuda()[:, 7:210], xs.cuda(), w.transpose(1, 2).contiguous().cuda().transpose(1, 2),
                                    ws.cuda()[..., None], off, None, b.cuda())
    assert torch.equal(got.cpu(), want)


@on_gpu
def test_grouped_empty(pkg):
    a, xs, w, ws, _ = grouped_inputs(16, 4, 2, 8, 32, "bf16", False)
    off = torch.zeros(3, dtype=torch.int32).cuda()
    f = pkg.ops.gemm_w8a8_grouped
    assert f(a[:0].cuda(), xs[:0].cuda(), w.cuda(), ws.cuda(), off).shape == (0, 8)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert f(a.cuda(), xs.cuda(), w.cuda(), ws.cuda(), off, none).shape == (0, 8)
    rows = torch.zeros(5, dtype=torch.int32, device="cuda")
    y = f(a[:0].cuda(), xs[:0].cuda(), w.cuda(), ws.cuda(), off + torch.tensor([0, 2, 5], device="cuda"), rows)
    assert y.shape == (5, 8) and (y == 0).all()


# ---------------------------------------------------------------------------
# 4-bit matrix-vector product
# ---------------------------------------------------------------------------


def matvec_inputs(seed, Rx, E, Nn, K, groups, dt, bias, sdt=torch.float32):
    g = gen(seed)
    lead = () if E is None else (E,)
    x = torch.randn(Rx, K, generator=g)
    x[:, torch.rand(K, generator=g) < 0.01] *= 20
    p = torch.randint(-128, 128, (*lead, Nn, K // 2), generator=g).to(torch.int8)
    s = torch.rand(*lead, Nn, *((K // 128,) if groups else ()), generator=g) * 8e-3 + 2e-3
    b = torch.randn(*lead, Nn, generator=g).to(TDT[dt]) if bias else None
    return x.to(TDT[dt]), p, s.to(sdt), b


def run_matvec(pkg, x, p, s, b, offsets=None, rows=None):
    c = lambda t: None if t is None else t.cuda()
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda()
    return pkg.ops.matvec_w4(c(x), c(p), c(s), c(b), off, c(rows))


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,Nn,K,groups,bias", [
    (1, 1, 2, False, False), (1, 16, 128, True, True), (2, 17, 256, True, False), (3, 100, 34, False, True),
    (5, 33, 130, False, True), (7, 129, 1440, False, False), (8, 64, 1024, True, True), (9, 48, 640, True, False),
    (16, 200, 384, True, True), (17, 31, 96, False, False), (33, 70, 2048, True, True), (70, 40, 512, True, False),
    (1, 2048, 8192, True, True), (4, 5, 16384, True, False), (1, 7, 20002, False, True)])
def test_matvec(pkg, dt, M, Nn, K, groups, bias):
    x, p, s, b = matvec_inputs(M + Nn + K, M, None, Nn, K, groups, dt, bias)
    got = run_matvec(pkg, x, p, s, b)
    assert got.dtype == TDT[dt] and got.shape == (M, Nn)
    assert_matvec(got, *matvec_ref(x, p, s, b, None, None), K)


@on_gpu
@pytest.mark.parametrize("K", [32000, 32256, 33024, 33408, 34048])
@pytest.mark.parametrize("M", [1, 3, 8])
def test_matvec_depth_at_the_limit_of_shared_memory(pkg, K, M):
    x, p, s, b = matvec_inputs(K, M, None, 40, K, True, "bf16", True)
    assert_matvec(run_matvec(pkg, x, p, s, b), *matvec_ref(x, p, s, b, None, None), K)


@on_gpu
@pytest.mark.parametrize("M,groups", [(1, True), (3, False), (6, True)])
def test_matvec_many_columns(pkg, M, groups):
    """Tiles of 64 rows, the last one partly filled; every 97th column and the last ones are looked at."""
    Nn, K = 56_900, 2048
    x, p, s, b = matvec_inputs(26, M, None, Nn, K, groups, "bf16", True)
    got = run_matvec(pkg, x, p, s, b).cpu()
    at = torch.cat((torch.arange(0, Nn - 80, 97), torch.arange(Nn - 80, Nn)))
    assert_matvec(got[:, at], *matvec_ref(x, p[at], s[at], b[at], None, None), K)


@on_gpu
@pytest.mark.parametrize("sdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [256, 384, 512, 1024, 2048, 4224])
@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_matvec_scales_of_any_alignment(pkg, sdt, K, off):
    """The scales come 16, 8, 4 or 2 bytes at a time."""
    x, p, s, b = matvec_inputs(27 + K, 5, 2, 70, K, True, "f16", True, sdt)
    room = torch.full((s.numel() + 8,), math.nan, dtype=sdt, device="cuda")
    view = room[off:off + s.numel()].view(s.shape)
    view.copy_(s)
    offsets = torch.tensor([0, 1, 5], dtype=torch.int32, device="cuda")
    got = pkg.ops.matvec_w4(x.cuda(), p.cuda(), view, b.cuda(), offsets)
    assert_matvec(got, *matvec_ref(x, p, s, b, [0, 1, 5], None), K)


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("off,pad", [(0, 0), (1, 0), (4, 4), (4, 1)])
def test_matvec_few_values_of_any_alignment(pkg, dt, off, pad):
    """Rows of x that begin at multiples of four values and others, in the call that makes its digits itself."""
    K = 1056
    x, p, s, b = matvec_inputs(28, 3, None, 90, K, False, dt, True)
    room = torch.full((off + 3 * (K + pad) + 4,), math.nan, dtype=x.dtype, device="cuda")
    view = room[off:off + 3 * (K + pad)].view(3, K + pad)[:, :K]
    view.copy_(x)
    assert_matvec(pkg.ops.matvec_w4(view, p.cuda(), s.cuda(), b.cuda()), *matvec_ref(x, p, s, b, None, None), K)
    rows = torch.tensor([2, -1, 0, 7, 2], dtype=torch.int32)
    got = pkg.ops.matvec_w4(view, p.cuda(), s.cuda(), b.cuda(), None, rows.cuda())
    assert_matvec(got, *matvec_ref(x, p, s, b, None, rows), K)


@on_gpu
@pytest.mark.parametrize("K", [256, 258])  # both kernels (258: one scale a row)
@pytest.mark.parametrize("xe,se", [(100, -120), (-110, 100), (0, -126), (127, -126)])
def test_matvec_scales_far_from_one(pkg, K, xe, se):
    x, p, s, _ = matvec_inputs(25, 3, None, 50, K, K == 256, "f32", False)
    x = torch.ldexp(x / x.abs().max() * 2.0 ** -8, torch.tensor(xe))
    s = torch.ldexp(s / s.max(), torch.tensor(se))
    s = s.clamp_min(torch.finfo(torch.float32).smallest_normal)
    assert_matvec(run_matvec(pkg, x, p, s, None), *matvec_ref(x, p, s, None, None, None), K)


@on_gpu
@pytest.mark.parametrize("dt,sdt", [("bf16", torch.bfloat16), ("f16", torch.float32), ("f32", torch.bfloat16)])
@pytest.mark.parametrize("counts,Nn,K,groups", [
    ([1], 40, 128, True), ([0, 3, 0, 1], 65, 256, True), ([2, 9, 40, 1], 24, 384, True), ([1] * 20, 128, 96, False),
    ([0] * 60 + [1, 0, 2], 33, 130, False)])
@pytest.mark.parametrize("gather", [False, True])
def test_matvec_experts(pkg, dt, sdt, counts, Nn, K, groups, gather):
    R, E = sum(counts), len(counts)
    Rx = max(1, R // 2) if gather else R
    x, p, s, b = matvec_inputs(R + Nn, Rx, E, Nn, K, groups, dt, True, sdt)
    rows = torch.randint(0, Rx, (R,), generator=gen(6)).to(torch.int32) if gather else None
    got = run_matvec(pkg, x, p, s, b, cum(counts), rows)
    assert_matvec(got, *matvec_ref(x, p, s, b, cum(counts), rows), K)


@on_gpu
@pytest.mark.parametrize("offsets", [[0, 4, 9, 9], [3, 10, 12, 20], [0, 0, 0, 0], [-7, 5, 2, 90], [0, 12, 3, 8],
                                     [40, 50, 60, 70], [2 ** 31 - 1, -2 ** 31, 0, 5]])
def test_matvec_any_offsets_are_safe(pkg, offsets):
    x, p, s, b = matvec_inputs(20, 24, 3, 40, 256, True, "bf16", True)
    rows = torch.randint(-3, 27, (24,), generator=gen(7)).to(torch.int32)
    got = run_matvec(pkg, x, p, s, b, offsets, rows)
    y, mag = matvec_ref(x, p, s, b, offsets, rows)
    assert_matvec(got, y, mag, 256)
    inside = torch.zeros(24, dtype=torch.bool)
    for lo, hi in spans(offsets, 24):
        inside[lo:hi] = True
    assert (got.cpu()[~inside] == 0).all()


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_matvec_every_code_exactly(pkg, dt):
    """Rows of one-hot activations return each weight's own value: codes -8
    to 7 in every nibble of every byte position, one scale 1."""
    K, Nn = 256, 48
    p = torch.arange(Nn * K // 2).mul(37).remainder(256).sub(128).to(torch.int8).reshape(Nn, K // 2)
    x = torch.eye(K)[:64].to(TDT[dt])
    got = run_matvec(pkg, x, p, torch.ones(Nn), None)
    assert torch.equal(got.cpu().double(), unpack(p)[:, :64].T)


@on_gpu
def test_matvec_layouts(pkg):
    x, p, s, b = matvec_inputs(21, 6, None, 50, 384, True, "bf16", True)
    want = run_matvec(pkg, x, p, s, b)
    wide = torch.zeros(6, 401, dtype=torch.bfloat16)
    for at in (0, 1, 8, 17):  # rows off any alignment
        wide[:, at:at + 384] = x
        got = pkg.ops.matvec_w4(wide.cuda()[:, at:at + 384], p.cuda(), s.cuda(), b.cuda())
        assert_matvec(got, *matvec_ref(x, p, s, b, None, None), 384)
    buf = torch.zeros(50 * 192 + 1, dtype=torch.int8).cuda()
    buf[1:] = p.cuda().reshape(-1)  # an odd base address
    got = pkg.ops.matvec_w4(x.cuda(), buf[1:].view(50, 192), s.cuda(), b.cuda())
    assert_matvec(got, *matvec_ref(x, p, s, b, None, None), 384)
    got = pkg.ops.matvec_w4(x.cuda(), p.cuda(), s.T.contiguous().cuda().T, b.cuda())
    assert torch.equal(got, want)
    half = s.to(torch.bfloat16)
    for at in (0, 1, 2, 3):  # two-byte scales off a word, three a row
        buf = torch.zeros(50 * 3 + 3, dtype=torch.bfloat16).cuda()
        buf[at:at + 150] = half.cuda().reshape(-1)
        got = pkg.ops.matvec_w4(x.cuda(), p.cuda(), buf[at:at + 150].view(50, 3), b.cuda())
        assert_matvec(got, *matvec_ref(x, p, half, b, None, None), 384)
    assert pkg.ops.matvec_w4(x[:0].cuda(), p.cuda(), s.cuda(), b.cuda()).shape == (0, 50)


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 3, 12])
def test_matvec_large_value_under_a_zero_weight(pkg, dt, M):
    """A value far above the others of its 128 k sets their unit, 2^-30 of it,
    also where its own weight is 0: half a unit of each of the 128 at most."""
    x, p, s, _ = matvec_inputs(24, M, None, 60, 384, True, dt, False)
    big = 2.0 ** 14
    x[:, 130] = big
    p[:, 65] &= -16  # the low nibble of k 130
    got = run_matvec(pkg, x, p, s, None)
    y, mag = matvec_ref(x, p, s, None, None, None)
    off = 2.0 ** -31 * 2 * big * (unpack(p)[:, 128:256].abs().sum(1) * s[:, 1].double())  # (e: below the next power of two)
    assert ((got.cpu().double() - y).abs() <= off + (384 / 16 + 3 + 40) * 2.0 ** -22 * mag
            + torch.finfo(TDT[dt]).eps / 2 * 1.001 * y.abs()).all()
    if dt == "bf16":  # exact down to 2^-22 of the largest: nothing is lost here but the usual
        near = x.abs() >= big * 2.0 ** -22
        x = torch.where(near, x, torch.zeros((), dtype=x.dtype))
        assert_matvec(run_matvec(pkg, x, p, s, None), *matvec_ref(x, p, s, None, None, None), 384)


@on_gpu
@pytest.mark.parametrize("K", [256, 130])  # both kernels
def test_matvec_non_finite_in_few_rows(pkg, K):
    x, p, s, b = matvec_inputs(23, 2, None, 70, K, False, "f32", True)
    x[0, 3], x[1, 5] = -math.inf, 2.0
    for rows in (None, torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1, 0, 1, 0, 0], dtype=torch.int32)):
        got = run_matvec(pkg, x, p, s, b, None, rows).cpu()
        y, mag = matvec_ref(x, p, s, b, None, rows)
        for r, src in enumerate([0, 1] if rows is None else rows.tolist()):
            if src == 1:
                assert_matvec(got[r:r + 1], y[r:r + 1], mag[r:r + 1], K)
            else:
                q = unpack(p)[:, 3]
                assert torch.equal(got[r].isnan(), q == 0) and (got[r][q > 0] == -math.inf).all()
                assert (got[r][q < 0] == math.inf).all()


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_matvec_non_finite_and_large(pkg, dt):
    """Infinities and NaN of a row stay in that row, and so do values near
    the type's largest (up to 1e36: the group's sum is taken before its
    scale)."""
    x, p, s, _ = matvec_inputs(22, 9, None, 40, 256, True, dt, False)
    x[2, 5], x[4, 7] = math.inf, math.nan
    x[6], x[6, 0] = 0.0, min(torch.finfo(TDT[dt]).max, 1e36)
    got = run_matvec(pkg, x, p, s, None).cpu()
    q = unpack(p)
    assert got[4].isnan().all()
    assert got[2].isinf()[q[:, 5] != 0].all() and got[2].isnan()[q[:, 5] == 0].all()
    y, mag = matvec_ref(x, p, s, None, None, None)
    keep = [0, 1, 3, 5, 7, 8]
    assert_matvec(got[keep], y[keep], mag[keep], 256)
    big = y[6]
    fits = big.abs() <= torch.finfo(TDT[dt]).max * 0.99
    assert_matvec(got[6][fits], big[fits], mag[6][fits], 256)


# ---------------------------------------------------------------------------
# combine
# ---------------------------------------------------------------------------


def check_combine(pkg, T, k, Nn, dt, residual, drop):
    R = T * k + 3
    y = randn(T, R, Nn).to(TDT[dt])
    w = torch.softmax(randn(T + 1, T, k), -1)
    pos = torch.randint(0, R, (T, k), generator=gen(8)).to(torch.int32)
    if drop:
        pos[torch.rand(T, k, generator=gen(9)) < 0.4] = -1
        pos[0] = torch.tensor([R, 2 ** 31 - 1, -2 ** 31, -5])[:k] if k <= 4 else R
    res = randn(T + 2, T, Nn).to(TDT[dt]) if residual else None
    got = pkg.ops.combine_experts(y.cuda(), w.cuda(), pos.cuda(), None if res is None else res.cuda()).cpu()
    ok = (pos >= 0) & (pos < R)
    terms = torch.where(ok, w, torch.zeros(())).double()[..., None] * y.double()[pos.clamp(0, R - 1).long()]
    want, mag = terms.sum(1), terms.abs().sum(1)
    if res is not None:
        want, mag = want + res.double(), mag + res.double().abs()
    # k multiply-adds and the residual's add, each half a float32 step of at
    # most the terms' magnitude; half a step of the result's dtype
    tol = (k + 1) * U * mag + torch.finfo(TDT[dt]).eps / 2 * 1.001 * want.abs() + \
        torch.finfo(TDT[dt]).smallest_normal * torch.finfo(TDT[dt]).eps
    assert ((got.double() - want).abs() <= tol).all()


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,k,Nn,residual,drop", [(1, 1, 1, False, False), (1, 8, 4096, False, False),
                                                  (5, 3, 100, True, True), (37, 2, 1025, True, False),
                                                  (300, 4, 64, False, True), (9, 32, 520, True, True)])
def test_combine(pkg, T, k, Nn, dt, residual, drop):
    check_combine(pkg, T, k, Nn, dt, residual, drop)


@on_gpu
def test_combine_layouts_and_empty(pkg):
    y = randn(30, 20, 96).to(torch.bfloat16).cuda()
    w, pos = torch.rand(5, 2, device="cuda"), torch.randint(0, 20, (5, 2), device="cuda")
    res = randn(31, 5, 96).to(torch.bfloat16).cuda()
    want = pkg.ops.combine_experts(y, w, pos, res)
    wide = torch.zeros(20, 200, dtype=torch.bfloat16, device="cuda")
    for at in (0, 3, 8):
        wide[:, at:at + 96] = y
        assert torch.equal(pkg.ops.combine_experts(wide[:, at:at + 96], w, pos.T.contiguous().T, res), want)
    none = torch.full((5, 2), -1, device="cuda")
    assert torch.equal(pkg.ops.combine_experts(y, w, none, res), res)
    assert (pkg.ops.combine_experts(y, w, none) == 0).all()
    assert (pkg.ops.combine_experts(y[:0], w, none) == 0).all()
    assert pkg.ops.combine_experts(y, w[:0], pos[:0]).shape == (0, 96)
    # NaN and infinities in rows that no token takes do not get in
    y[7] = math.nan
    y[8] = math.inf
    assert torch.isfinite(pkg.ops.combine_experts(y, w, torch.where((pos == 7) | (pos == 8), -1, pos), res)).all()


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------


def situ64(h):
    a, b = h.chunk(2, -1)
    return 4 * torch.tanh(b / 4) * torch.sigmoid(b) * 25 * torch.tanh(a / 25)


@on_gpu
@pytest.mark.parametrize("T", [1, 5, 150])
@pytest.mark.parametrize("rot", [None, ("regular", 64)])
def test_int8_feed_forward_is_its_operators(pkg, T, rot):
    """The composed call against the same steps expert by expert with the
    dense operators: bit for bit up to the float32 sum, which the plain
    float64 sum of the same rows bounds."""
    E, k, K, F = 6, 2, 256, 128
    x = randn(40, T, K).to(torch.bfloat16).cuda()
    logits = randn(41, T, E).cuda()
    X = pkg.experts
    up, us = X.quantize_experts_int8(randn(42, E, 2 * F, K).cuda() * 0.05, rot)
    down, ds = X.quantize_experts_int8(randn(43, E, K, F).cuda() * 0.05, rot)
    res = randn(44, T, K).to(torch.bfloat16).cuda()
    got = X.int8_forward_experts(x.reshape(1, T, K), logits.reshape(1, T, E), up, us, down, ds, k, residual=res,
                                 rot=rot, down_rot=rot)
    assert got.shape == (1, T, K)
    ids, w, *_ = pkg.ops.route_experts(logits, k)
    want, mag = res.double(), res.double().abs()
    xq, xs = pkg.ops.quant_act_int8(x, rot)
    for e in range(E):
        h = pkg.ops.gemm_w8a8(xq, xs, up[e], us[e])
        y = pkg.ops.gemm_w8a8(*pkg.ops.quant_act_int8(pkg.ops.situ(h), rot), down[e], ds[e]).double()
        we = (w.double() * (ids == e)).sum(1, keepdim=True)
        want, mag = want + we * y, mag + (we * y).abs()
    tol = (k + 1) * U * mag + 2.0 ** -8 * 1.001 * want.abs()
    assert ((got.reshape(T, K).double() - want).abs() <= tol).all()


@on_gpu
@pytest.mark.parametrize("T,group,rot", [(1, 128, None), (3, 0, ("regular", 64)), (20, 128, ("sylvester", 128))])
def test_w4_feed_forward(pkg, T, group, rot):
    """Against the dequantised weights in float64, float32 activations, so
    that no rounding to 16 bits hides an error.  A product of 256 terms is
    within (256/16 + 2 + 40) * 2^-22 = 1.4e-5 of its terms' magnitude
    (assert_matvec), which is about sqrt(256) = 16 times the sum's own size:
    2.2e-4 of it.  Two products, and a few float32 steps of the activation
    and the rotations: 5e-4 of the largest value."""
    E, k, K, F = 5, 2, 256, 256
    x, logits = randn(50, T, K), randn(51, T, E)
    X = pkg.experts
    up, us = X.quantize_experts_int4(randn(52, E, 2 * F, K).cuda() * 0.05, rot, group)
    down, ds = X.quantize_experts_int4(randn(53, E, K, F).cuda() * 0.05, rot, group)
    got = X.w4_forward_experts(x.cuda(), logits.cuda(), up, us, down, ds, k, rot=rot, down_rot=rot).cpu().double()

    def weight(p, s):
        q = unpack(p.cpu())
        s = s.cpu().double()
        return q * (s.repeat_interleave(128, -1) if group else s[..., None])

    def rotated(v):
        return v.double() if rot is None else pkg.ops.rotate(v.float().cuda(), *rot).cpu().double()

    wu, wd = weight(up, us), weight(down, ds)
    ids, w, *_ = route_ref(logits, k, "softmax", True)
    want = torch.zeros(T, K, dtype=torch.float64)
    xr = rotated(x)
    for t in range(T):
        for j in range(k):
            h = situ64(xr[t] @ wu[ids[t, j]].T)
            want[t] += w[t, j] * (rotated(h[None])[0] @ wd[ids[t, j]].T)
    assert (got - want).abs().max() <= 5e-4 * want.abs().max()


@on_gpu
@pytest.mark.parametrize("group", [0, 128])
def test_convrot_w4a16_forward(pkg, group):
    w = randn(60, 96, 512).cuda() * 0.02
    x = randn(61, 2, 3, 512).to(torch.bfloat16).cuda()
    b = randn(62, 96).to(torch.bfloat16).cuda()
    p, s = pkg.ops.quant_weight_int4(w, ("regular", 256), group)
    y = pkg.int4_quant.convrot_w4a16_forward(x, p, s, b, 256, torch.bfloat16)
    assert y.shape == (2, 3, 96)
    xr = pkg.ops.rotate(x.reshape(6, 512), "regular", 256)
    assert_matvec(y.reshape(6, 96), *matvec_ref(xr.cpu(), p.cpu(), s.cpu(), b.cpu(), None, None), 512)
    with pytest.raises(ValueError):
        pkg.int4_quant.convrot_w4a16_forward(x[..., :256], p, s, b, 256, torch.bfloat16)


def layer(pkg, seed, T, dt=torch.bfloat16):
    E, k, K, F = 8, 2, 256, 128
    X = pkg.experts
    u, us = X.quantize_experts_int8(randn(seed, E, 2 * F, K).cuda() * 0.05)
    d, ds = X.quantize_experts_int8(randn(seed + 1, E, K, F).cuda() * 0.05)
    u4, us4 = X.quantize_experts_int4(randn(seed, E, 2 * F, K).cuda() * 0.05, None, 128)
    d4, ds4 = X.quantize_experts_int4(randn(seed + 1, E, K, F).cuda() * 0.05, None, 128)
    x, logits = randn(seed + 2, T, K).to(dt).cuda(), randn(seed + 3, T, E).cuda()
    return x, logits, lambda: (X.int8_forward_experts(x, logits, u, us, d, ds, k),
                               X.w4_forward_experts(x, logits, u4, us4, d4, ds4, k))


@on_gpu
@pytest.mark.parametrize("T", [1, 200])
def test_graph_replay_follows_new_inputs(pkg, T):
    """Captured once, replayed on other tokens with other experts; a second
    graph of the same layer replayed in between shares nothing with it."""
    x, logits, f = layer(pkg, 70, T)
    f()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for turn in range(3):
        x.copy_(randn(80 + turn, *x.shape))
        logits.copy_(randn(90 + turn, *logits.shape) * (turn + 1))
        want = f()
        for i in (0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)
    assert pkg.ops.device_error() == 0


@on_gpu
def test_two_streams_at_once(pkg):
    calls = [layer(pkg, 100 + 10 * i, 300) for i in range(2)]
    want = [c[2]() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls[i][2]())
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            for a, b in zip(pair, want[i]):
                assert torch.equal(a, b)


@on_gpu
def test_results_repeat(pkg):
    x, logits, f = layer(pkg, 130, 777)
    first = f()
    for _ in range(5):
        for a, b in zip(f(), first):
            assert torch.equal(a, b)


@on_gpu
def test_opcheck(pkg):
    ns = torch.ops.qlin_b200
    utils = ("test_schema", "test_faketensor")
    logits = randn(140, 9, 6).cuda()
    torch.library.opcheck(ns.route_experts.default, (logits, 2, "softmax", True), test_utils=utils)
    ids, w, off, rows, pos = pkg.ops.route_experts(logits, 2)
    a, xs, wq, ws, b = [t.cuda() for t in grouped_inputs(141, 9, 6, 24, 64, "bf16", True)]
    torch.library.opcheck(ns.gemm_w8a8_grouped.default, (a, xs, wq, ws, off, rows, b, torch.bfloat16),
                          test_utils=utils)
    x, p, s, b4 = [t.cuda() for t in matvec_inputs(142, 9, 6, 24, 128, True, "bf16", True)]
    torch.library.opcheck(ns.matvec_w4.default, (x, p, s, b4, off, rows), test_utils=utils)
    y = randn(143, 18, 24).cuda()
    torch.library.opcheck(ns.combine_experts.default, (y, w, pos, None), test_utils=utils)


@on_gpu
def test_compiled_feed_forward(pkg):
    x, logits, f = layer(pkg, 150, 40)
    torch._dynamo.reset()
    for a, b in zip(torch.compile(f, fullgraph=True)(), f()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# CPU: fakes and refusals
# ---------------------------------------------------------------------------


def test_registered_with_fake_shapes(pkg):
    L = pkg.library
    d = dict(device="cuda")
    with FakeTensorMode():
        ids, w, off, rows, pos = L.route_experts(torch.empty(10, 6, dtype=torch.bfloat16, **d), 2)
        assert ids.shape == w.shape == pos.shape == (10, 2) and off.shape == (7,) and rows.shape == (20,)
        assert w.dtype == torch.float32 and {ids.dtype, off.dtype, rows.dtype, pos.dtype} == {torch.int32}
        a, wq = torch.empty(10, 64, dtype=torch.int8, **d), torch.empty(6, 24, 64, dtype=torch.int8, **d)
        xs, ws = torch.empty(10, 1, **d), torch.empty(6, 24, **d)
        y = L.gemm_w8a8_grouped(a, xs, wq, ws, off, rows, None, torch.float16)
        assert (y.shape, y.dtype) == ((20, 24), torch.float16)
        assert L.gemm_w8a8_grouped(a, xs, wq, ws, off).shape == (10, 24)
        x = torch.empty(10, 128, dtype=torch.bfloat16, **d)
        y = L.matvec_w4(x, wq, torch.empty(6, 24, 1, **d), None, off, rows)
        assert (y.shape, y.dtype) == ((20, 24), torch.bfloat16)
        assert L.matvec_w4(x, wq[0], ws[0]).shape == (10, 24)
        assert L.combine_experts(y, w, pos).shape == (10, 24)
    for name in ("route_experts", "combine_experts", "gemm_w8a8_grouped", "matvec_w4"):
        assert torch._library.utils.has_fake_kernel(getattr(torch.ops.qlin_b200, name).default)


def test_python_refusals(pkg):
    """Raised before anything is launched or a device is asked for."""
    o = pkg.ops
    lg = torch.zeros(4, 6)
    for bad in (lambda: o.route_experts(lg[0], 2), lambda: o.route_experts(lg, 0), lambda: o.route_experts(lg, 7),
                lambda: o.route_experts(lg, 2, "tanh"), lambda: o.route_experts(torch.zeros(4, 513), 2),
                lambda: o.route_experts(torch.zeros(4, 64), 33), lambda: o.route_experts(torch.zeros(4, 0), 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        o.route_experts(lg.int(), 2)
    a, w = torch.zeros(5, 32, dtype=torch.int8), torch.zeros(2, 8, 32, dtype=torch.int8)
    xs, ws, off = torch.ones(5, 1), torch.ones(2, 8), torch.tensor([0, 2, 5], dtype=torch.int32)
    g = o.gemm_w8a8_grouped
    for bad in (lambda: g(a, xs, w[0], ws, off), lambda: g(a[:, :16], xs, w, ws, off), lambda: g(a, xs, w, ws, off[:2]),
                lambda: g(a, xs[:4], w, ws, off), lambda: g(a, xs, w, ws[:, :7], off), lambda: g(a, xs, w, ws.T, off),
                lambda: g(a, xs, w, ws, off, off[None]), lambda: g(a, xs, w, ws, off, None, ws[0]),
                lambda: g(a, xs, w[:0], ws[:0], off[:1]), lambda: g(a, xs, w.to("meta"), ws, off)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: g(a.float(), xs, w, ws, off), lambda: g(a, xs, w, ws, off.float()),
                lambda: g(a, xs, w, ws, off, None, None, torch.float64)):
        with pytest.raises(TypeError):
            bad()
    x, p, s = torch.zeros(3, 256), torch.zeros(10, 128, dtype=torch.int8), torch.ones(10, 2)
    m = o.matvec_w4
    for bad in (lambda: m(x[:, :128], p, s), lambda: m(x, p, s[:, :1].expand(10, 3)), lambda: m(x, p[None], s),
                lambda: m(x, p, s, None, off), lambda: m(x, p, s[:9]), lambda: m(x, p, s, torch.zeros(9)),
                lambda: m(x[0], p, s), lambda: m(x, p, s, None, None, off[None])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: m(x, p.int(), s), lambda: m(x.double(), p, s), lambda: m(x, p, s, None, None, s[0])):
        with pytest.raises(TypeError):
            bad()
    y, wt, pos = torch.zeros(6, 16), torch.ones(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    for bad in (lambda: o.combine_experts(y, wt[:2], pos), lambda: o.combine_experts(y, wt, pos[0]),
                lambda: o.combine_experts(y, wt, pos, torch.zeros(3, 15)), lambda: o.combine_experts(y[0], wt, pos),
                lambda: o.combine_experts(y, wt, pos, torch.zeros(3, 16, dtype=torch.float16)),
                lambda: o.combine_experts(y, wt[:, :0], pos[:, :0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        o.combine_experts(y, wt, wt)
    for call in (lambda: o.route_experts(lg, 2), lambda: g(a, xs, w, ws, off), lambda: m(x, p, s),
                 lambda: o.combine_experts(y, wt, pos)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="tokens"):
        pkg.experts.int8_forward_experts(torch.zeros(4, 32), torch.zeros(3, 2), w, ws, w, ws, 1)


def test_abi_refusals(pkg):
    """Status codes of the C entry points; none of these calls reaches a device."""
    N = pkg._native
    lib = N.load()
    bad, align, unsup = N.ERR_INVALID_ARG, N.ERR_ALIGNMENT, N.ERR_UNSUPPORTED
    route = lambda dt=N.F32, T=4, E=6, ld=6, k=2, sc=0, off=16: lib.qlin_route_experts(
        16, dt, T, E, ld, k, sc, 1, 16, 16, off, 16, 16, None, 0, None)
    assert route(E=0) == route(E=513, ld=513) == route(ld=5) == route(k=0) == route(k=7) == route(T=-1) == bad
    assert route(dt=9) == route(sc=2) == route(off=None) == bad
    assert route(T=2 ** 31 - 1) == unsup
    assert route(T=1000) == bad and b"workspace" in lib.qlin_last_error()
    import ctypes
    n = ctypes.c_uint64(7)
    assert lib.qlin_route_experts_workspace(1, 8, ctypes.addressof(n)) == 0 and n.value == 0
    assert lib.qlin_route_experts_workspace(100000, 9, ctypes.addressof(n)) == 0 and n.value > 0 and n.value % 16 == 0
    assert lib.qlin_route_experts_workspace(0, 8, ctypes.addressof(n)) == 0 and n.value == 0
    assert lib.qlin_route_experts_workspace(1, 0, ctypes.addressof(n)) == bad
    assert lib.qlin_route_experts_workspace(1, 8, None) == bad
    comb = lambda y=16, R=4, Nn=8, ld=8, T=2, k=2, res=None, ldr=8, dt=N.BF16: lib.qlin_combine_experts(
        y, dt, R, Nn, ld, 16, 16, T, k, res, ldr, 16, None)
    assert comb(ld=7) == comb(k=0) == comb(T=-1) == comb(res=16, ldr=7) == comb(dt=N.I8) == comb(y=None) == bad
    assert comb(T=0) == comb(Nn=0, ld=0) == 0
    grp = lambda Ra=4, E=2, R=4, Nn=8, K=32, rows=None, off=16, dt=N.BF16, a=16, out=16, ws=None, nws=0: lib.qlin_gemm_w8a8_grouped(
        a, 16, Ra, 16, 16, off, E, rows, None, out, dt, R, Nn, K, ws, nws, None)
    assert grp(E=0) == grp(E=513) == grp(R=5) == grp(K=0) == grp(Nn=-1) == grp(off=None) == grp(dt=N.I8) == bad
    assert grp(K=20) == grp(a=24) == grp(out=20) == align
    assert grp(K=131072) == grp(E=512, Nn=2 ** 23) == unsup
    assert grp(R=0, Ra=0) == grp(Nn=0) == 0
    assert lib.qlin_gemm_w8a8_grouped_workspace(4, 32, ctypes.addressof(n)) == 0 and n.value >= 4 * 32 + 4 * 4
    assert lib.qlin_gemm_w8a8_grouped_workspace(-1, 32, ctypes.addressof(n)) == bad
    assert grp(rows=16) == grp(rows=16, ws=16, nws=n.value - 16) == bad
    assert grp(rows=16, ws=8, nws=4096) == align
    mv = lambda Rx=4, ld=256, sdt=N.F32, group=128, off=None, E=1, R=4, Nn=8, K=256, dt=N.BF16, x=16, ws=16, nws=2 ** 20, out=16: lib.qlin_matvec_w4(
        x, dt, Rx, ld, 16, 16, sdt, group, off, E, None, None, out, R, Nn, K, ws, nws, None)
    assert mv(E=2) == mv(E=513, off=16) == mv(R=3) == mv(K=255) == mv(ld=255) == mv(sdt=N.F16) == mv(dt=N.I8) == bad
    assert mv(K=250, ld=250) == mv(x=None) == bad
    assert mv(group=64) == mv(E=512, off=16, Nn=2 ** 23) == unsup
    assert mv(R=0, Rx=0) == mv(Nn=0) == 0
    assert lib.qlin_matvec_w4_workspace(16, 0, 40, 40, 8, 256, ctypes.addressof(n)) == 0 and n.value >= 40 * 256 * 4
    assert mv(R=40, Rx=40, ws=None) == mv(R=40, Rx=40, nws=n.value - 1) == bad
    assert mv(ws=24) == mv(out=24) == align
    assert lib.qlin_matvec_w4_workspace(16, 0, -1, 4, 8, 256, ctypes.addressof(n)) == bad
    assert lib.qlin_matvec_w4_workspace(16, 0, 1, 1, 8, 256, ctypes.addressof(n)) == 0 and n.value == 0
    assert lib.qlin_matvec_w4_workspace(17, 0, 1, 1, 8, 256, ctypes.addressof(n)) == 0 and n.value > 0
    assert lib.qlin_matvec_w4_workspace(16, 1, 1, 1, 8, 256, ctypes.addressof(n)) == 0 and n.value > 0


def test_matvec_stall_refusals(pkg):
    N = pkg._native
    lib = N.load()
    bad, align, unsup = N.ERR_INVALID_ARG, N.ERR_ALIGNMENT, N.ERR_UNSUPPORTED
    st = lambda x=16, w=16, R=40, Nn=8, K=256, group=128, ws=16, nws=2 ** 20, which=0, stage=0: \
        lib.qlin_selftest_matvec_stall(x, w, 16, group, 16, R, Nn, K, ws, nws, which, stage, None)
    assert st(x=None) == st(R=0) == st(Nn=0) == st(K=0) == st(K=16512) == st(K=160) == st(K=48, group=0) == bad
    assert st(which=-1) == st(stage=-1) == st(ws=None) == st(nws=40 * 256) == bad
    assert st(group=64) == unsup
    assert st(w=24) == st(ws=24) == align
    assert st(which=1, group=0) == st(which=2) == bad


def test_grouped_stall_refusals(pkg):
    N = pkg._native
    lib = N.load()
    bad, align = N.ERR_INVALID_ARG, N.ERR_ALIGNMENT
    st = lambda a=16, E=2, R=4, Nn=8, K=32, which=0, stage=0, off=16: \
        lib.qlin_selftest_grouped_stall(a, 16, 16, 16, off, E, 16, R, Nn, K, which, stage, None)
    assert st(a=None) == st(E=0) == st(E=513) == st(R=0) == st(Nn=0) == st(K=0) == st(K=131072) == st(off=None) == bad
    assert st(which=-1) == st(which=3) == st(stage=-1) == st(E=512, Nn=2 ** 23) == bad
    assert st(K=40) == st(a=24) == align


@pytest.mark.parametrize("aligned", [True, False])
def test_matvec_workspace_goes_by_the_fewer_rows(pkg, aligned):
    """Few rows gathered out of a long x need no more room than those rows by themselves."""
    import ctypes
    lib, n = pkg._native.load(), ctypes.c_uint64(0)

    def room(R, Rx, K=4096):
        assert lib.qlin_matvec_w4_workspace(16 if aligned else 17, 1, R, Rx, 8, K, ctypes.addressof(n)) == 0
        return n.value

    assert 0 < room(8, 65536) == room(8, 8)
    assert room(65536, 8) == room(8, 8)
    assert room(0, 100) == room(100, 0) == 0


@on_gpu
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("K,groups", [(256, True), (2048, False), (258, False)])  # 258: the kernel for any depth
@pytest.mark.parametrize("E", [None, 5])
def test_matvec_few_rows_of_a_long_x(pkg, dt, K, groups, E):
    """The same bits as for those rows laid out one after another."""
    Rx, R = 700, 23
    x, p, s, b = matvec_inputs(29 + K, Rx, E, 70, K, groups, dt, True)
    x[5, 3], x[6, 7] = math.inf, math.nan
    rows = torch.randint(0, Rx, (R,), generator=gen(10)).to(torch.int32)
    rows[:6] = torch.tensor([5, 699, -1, 6, Rx, 699])
    offsets = None if E is None else [0, 1, 9, 9, 21, 22]
    got = run_matvec(pkg, x, p, s, b, offsets, rows)
    inside = (rows >= 0) & (rows < Rx)
    laid = torch.where(inside[:, None], x[rows.clamp(0, Rx - 1).long()], torch.zeros((), dtype=x.dtype))
    assert torch.equal(got.nan_to_num(nan=7.0), run_matvec(pkg, laid, p, s, b, offsets).nan_to_num(nan=7.0))
    good = torch.ones(R, dtype=torch.bool)
    good[[0, 3]] = False
    y, mag = matvec_ref(x.nan_to_num(0, 0, 0), p, s, b, offsets, rows)
    assert_matvec(got[good.cuda()], y[good], mag[good], K)


@pytest.mark.parametrize("lead", [(0,), (2, 0), (3,), (2, 3)])
def test_feed_forward_tokens_and_residual(pkg, lead):
    """Tokens, logits and residual as rows, also where there are none."""
    x, logits, res = torch.zeros(*lead, 32), torch.zeros(*lead, 4), torch.zeros(*lead, 24)
    T = math.prod(lead)
    x2, l2, r2 = pkg.experts._tokens(x, logits, res)
    assert (x2.shape, l2.shape, r2.shape) == ((T, 32), (T, 4), (T, 24))
    assert pkg.experts._tokens(x, logits, None)[2] is None


@on_gpu
@pytest.mark.parametrize("lead", [(0,), (2, 0)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rot", [None, ("regular", 64)])
def test_feed_forward_without_tokens(pkg, lead, residual, rot):
    E, K, F = 3, 128, 64
    X, bf = pkg.experts, dict(dtype=torch.bfloat16, device="cuda")
    x, logits = torch.zeros(*lead, K, **bf), torch.zeros(*lead, E, **bf)
    res = torch.zeros(*lead, K, **bf) if residual else None
    up, down = randn(160, E, 2 * F, K).cuda(), randn(161, E, K, F).cuda()
    y = X.int8_forward_experts(x, logits, *X.quantize_experts_int8(up, rot), *X.quantize_experts_int8(down, rot), 2,
                               residual=res, rot=rot, down_rot=rot)
    assert (y.shape, y.dtype) == (x.shape, x.dtype)
    y = X.w4_forward_experts(x, logits, *X.quantize_experts_int4(up, rot), *X.quantize_experts_int4(down, rot), 2,
                             residual=res, rot=rot, down_rot=rot)
    assert (y.shape, y.dtype) == (x.shape, x.dtype)


def assert_matvec_closely(got, x, p, s, bias=None, offsets=None, rows=None):
    """What the digits and float32 steps of the kernels may do.  Per 128 k: x
    as integers in units of 2^(e - 29), e the exponent of their largest, each
    off by half a unit at most; the digits' integer sums are exact, and their
    two halves (whose magnitudes add up to the terms' and less than 2^-12 of
    the largest x times the weights) each become a float32 and meet the scale,
    two steps.  Then a multiply-add for each 128 k, the halves' sum, eight
    warps' sums, the scale of a row and the bias: K / 128 + 13 steps of 2^-24
    of the magnitude; last, half a step of the result's dtype."""
    dt, K = got.dtype, x.shape[1]
    y, mag = matvec_ref(x, p, s, bias, offsets, rows)
    q = unpack(p).abs()
    blocks = -(-K // 128)
    pad = blocks * 128 - K
    big = torch.nn.functional.pad(x.double().abs(), (0, pad)).reshape(-1, blocks, 128).amax(-1)
    e = torch.where(big > 0, torch.frexp(big).exponent - 1, -126).clamp_min(-126)  # 2^e <= big < 2^(e + 1)
    qs = torch.nn.functional.pad(q, (0, pad)).reshape(*q.shape[:-1], blocks, 128).sum(-1)
    qs = qs * (s.double() if s.dim() == p.dim() and s.shape[-1] != 1 else s.double().reshape(*p.shape[:-1], 1))
    src = torch.arange(x.shape[0]) if rows is None else rows.long()
    inside = (src >= 0) & (src < x.shape[0])
    unit = torch.where(inside[:, None], torch.exp2((e - 30).double())[src.clamp(0, x.shape[0] - 1)], 0.0)
    off = torch.zeros_like(y)
    for i, (b, t) in enumerate([(0, len(src))] if offsets is None else spans(offsets, len(src))):
        off[b:t] = unit[b:t] @ (qs if offsets is None else qs[i]).T
    tol = off * 1.01 + (K / 128 + 13) * U * 1.001 * (mag + off * 2 ** 18) + torch.finfo(dt).eps / 2 * 1.001 * y.abs() + \
        torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ((got.cpu().double() - y).abs() > tol).sum().item()
    assert bad == 0, f"{bad} of {y.numel()} values off"


@on_gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M,Nn,K,groups", [
    (1, 300, 128, True), (1, 2048, 8192, True), (2, 129, 4224, False), (3, 200, 2048, True), (4, 100, 16384, True),
    (8, 70, 1440, False), (9, 640, 1024, True), (33, 70, 2048, True),
    (1, 33, 34, False), (3, 100, 258, False), (7, 50, 20002, False), (2, 40, 33408, True)])  # the kernel for any depth
def test_matvec_closely(pkg, dt, M, Nn, K, groups):
    x, p, s, b = matvec_inputs(30 + M + K, M, None, Nn, K, groups, dt, True)
    assert_matvec_closely(run_matvec(pkg, x, p, s, b), x, p, s, b)


@on_gpu
@pytest.mark.parametrize("K,groups", [(384, True), (416, False), (386, False)])  # 386: the kernel for any depth
@pytest.mark.parametrize("counts", [[1], [0, 3, 9, 1]])
def test_matvec_experts_closely_with_a_large_value_under_zero_weights(pkg, K, groups, counts):
    """A value 2^14 and more above the others sets the unit of its 128 k where its own weight is 0."""
    R, E = sum(counts), len(counts)
    x, p, s, b = matvec_inputs(31 + K, R, E, 60, K, groups, "f32", True)
    x[:, 130] = 2.0 ** 17
    p[:, :, 65] &= -16  # the low nibble of k 130
    rows = torch.randint(-1, R + 1, (R,), generator=gen(11)).to(torch.int32)
    for r in (None, rows):
        assert_matvec_closely(run_matvec(pkg, x, p, s, b, cum(counts), r), x, p, s, b, cum(counts), r)


@on_gpu
@pytest.mark.parametrize("M", [40, 200])
def test_matvec_rows_of_zeros_and_others_in_turn(pkg, M):
    """A row of zeros and a row of x at the same place of one pass after another."""
    x, p, s, b = matvec_inputs(32, 9, None, 4500, 2048, True, "bf16", True)
    rows = torch.randint(0, 9, (M,), generator=gen(12)).to(torch.int32)
    rows[torch.arange(M) // 8 % 2 == 0] = -1
    rows[torch.arange(M) % 5 == 0] = 9
    got = run_matvec(pkg, x, p, s, b, None, rows).cpu()
    at = torch.arange(0, 4500, 31)
    inside = (rows >= 0) & (rows < 9)
    assert torch.equal(got[~inside], b[None].expand(int((~inside).sum()), -1))
    assert_matvec_closely(got[:, at], x, p[at], s[at], b[at], None, rows)
