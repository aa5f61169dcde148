"""Failure detection on the GPU without a fault: bounded pipeline waits that
are made to run out return an error status the host reads, and the context
stays usable (a normal GEMM afterwards is still bit-exact).

The wait limit is lowered to a few milliseconds for these tests and restored
to its default afterwards.  Nothing here faults, traps or hangs a GPU: every
wait that runs out is a bounded loop that gives up after the limit.
"""
import numpy as np
import pytest
import torch

import golden_inputs as gi
from conftest import cuda_ok
from oracle import qlinear_oracle as O

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


@pytest.fixture
def short_limit(pkg):
    torch.cuda.synchronize()
    assert pkg.ops.device_error() == 0
    pkg.ops.set_wait_limit(5_000_000)  # 5 ms
    yield pkg
    pkg.ops.set_wait_limit(0)
    pkg.ops.device_error()


def _linear(P, M, N, K, seed):
    x = gi.activation(seed, M, K, "bf16")
    w = gi.weight(seed, N, K)
    wq, ws = O.quantize_int8_axiswise(w, 1)
    xq, xs = P.ops.quant_act_int8(torch.from_numpy(x).to(torch.bfloat16).cuda())
    return x, wq, ws, xq, xs


def _check_normal_gemm(P):
    x, wq, ws, xq, xs = _linear(P, 300, 520, 512, 41)
    y = P.ops.gemm_w8a8(xq, xs, torch.from_numpy(wq).cuda(), torch.from_numpy(ws).cuda(), None, torch.bfloat16)
    yo = O.int8_forward_dynamic_per_row(x, wq, ws, None, "bf16")
    np.testing.assert_array_equal(y.cpu().view(torch.int16).numpy().view(np.uint16), O.f32_to_bf16_bits(yo))
    assert P.ops.device_error() == 0


@pytest.mark.parametrize("which,bit", [(0, 1), (1, 2)])
def test_wait_selftest_times_out(short_limit, which, bit):
    P = short_limit
    P.ops.selftest_wait_timeout(which)
    torch.cuda.synchronize()
    assert P.ops.device_error() == bit
    _check_normal_gemm(P)


@pytest.mark.parametrize("M,N,K,stall_kb", [(512, 512, 1024, 3),  # CTA-pair kernel, all CTAs stall
                                            (128, 200, 512, 0)])  # single-CTA kernel
def test_gemm_stall_aborts_and_recovers(short_limit, M, N, K, stall_kb):
    P = short_limit
    _, wq, ws, xq, xs = _linear(P, M, N, K, 42)
    P.ops.selftest_gemm_stall(xq, xs, torch.from_numpy(wq).cuda(), torch.from_numpy(ws).cuda(), stall_kb)
    torch.cuda.synchronize()
    bits = P.ops.device_error()
    assert bits & 1, bits
    assert not bits & 4, bits  # the abort drained its in-flight loads and MMAs
    _check_normal_gemm(P)


def test_set_wait_limit_rejects_out_of_range(pkg):
    from comfyui_int8_fast_rocm_b200._native import NativeError
    with pytest.raises(NativeError):
        pkg.ops.set_wait_limit(10)  # below 1 us
    with pytest.raises(NativeError):
        pkg.ops.set_wait_limit(120 * 10**9)


def _matvec(P, R, N, K, grouped, seed=43):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g).to(torch.bfloat16).cuda()
    p = torch.randint(-128, 128, (N, K // 2), generator=g).to(torch.int8).cuda()
    s = (torch.rand(N, K // 128, generator=g) if grouped else torch.rand(N, generator=g)).cuda()
    return x, p, s


# rows of one, two and four column blocks, digits made in the kernel (R * K <= 8192) and before it
@pytest.mark.parametrize("R,K,stage", [(1, 1024, 0), (1, 8192, 2), (2, 16384, 3), (4, 4096, 1), (8, 2048, 0), (20, 4096, 5)])
@pytest.mark.parametrize("grouped", [False, True])
def test_matvec_stall_aborts_and_recovers(short_limit, R, K, stage, grouped):
    P, N = short_limit, 9000
    x, p, s = _matvec(P, R, N, K, grouped)
    want = P.ops.matvec_w4(x, p, s)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
    P.ops.selftest_matvec_stall(x, p, s, 0, stage)
    torch.cuda.synchronize()
    bits = P.ops.device_error()
    assert bits & 1, bits
    assert not bits & 4, bits  # the loads in flight were waited for
    assert torch.equal(P.ops.matvec_w4(x, p, s), want)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0


@pytest.mark.parametrize("R,K,stage", [(1, 1024, 0), (1, 8192, 1), (4, 16384, 2), (8, 4096, 0), (20, 8192, 9)])
def test_matvec_scales_giving_up_leaves_no_load_in_flight(short_limit, R, K, stage):
    """The producer goes on filling the ring after the scales' warp has left;
    its wait for those loads ends with them, not with the limit."""
    P, N = short_limit, 9000
    x, p, s = _matvec(P, R, N, K, True, 44)
    want = P.ops.matvec_w4(x, p, s)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
    P.ops.selftest_matvec_stall(x, p, s, 1, stage)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 1
    assert torch.equal(P.ops.matvec_w4(x, p, s), want)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0


def _grouped(P, counts, N, K, seed=45):
    g = torch.Generator().manual_seed(seed)
    R, E = sum(counts), len(counts)
    a = torch.randint(-127, 128, (R, K), generator=g).to(torch.int8).cuda()
    w = torch.randint(-127, 128, (E, N, K), generator=g).to(torch.int8).cuda()
    off = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32).cuda()
    return a, torch.rand(R, 1, generator=g).cuda() * 1e-2, w, torch.rand(E, N, generator=g).cuda() * 1e-3, off


GROUPED_STALLS = [([1], 200, 512, 1), ([300, 5, 700], 1000, 2048, 7), ([3, 0, 40], 600, 1328, 4),
                  ([2000, 90] * 8, 2048, 1024, 13), ([2000, 90] * 8, 2048, 1024, 0)]


@pytest.mark.parametrize("counts,N,K,stage", GROUPED_STALLS)
def test_grouped_stall_aborts_and_recovers(short_limit, counts, N, K, stage):
    P = short_limit
    a, xs, w, ws, off = _grouped(P, counts, N, K)
    want = P.ops.gemm_w8a8_grouped(a, xs, w, ws, off)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
    P.ops.selftest_grouped_stall(a, xs, w, ws, off, 0, stage)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 1
    assert torch.equal(P.ops.gemm_w8a8_grouped(a, xs, w, ws, off), want)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
    _check_normal_gemm(P)


@pytest.mark.parametrize("which", [1, 2])
@pytest.mark.parametrize("counts,N,K,stage", GROUPED_STALLS)
def test_grouped_one_producer_giving_up_leaves_no_load_in_flight(short_limit, counts, N, K, stage, which):
    """The other producer of the pair goes on filling the ring; both end with
    as many stages filled, and the leader awaits all of them."""
    P = short_limit
    a, xs, w, ws, off = _grouped(P, counts, N, K, 46)
    want = P.ops.gemm_w8a8_grouped(a, xs, w, ws, off)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
    P.ops.selftest_grouped_stall(a, xs, w, ws, off, which, stage)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 1
    assert torch.equal(P.ops.gemm_w8a8_grouped(a, xs, w, ws, off), want)
    torch.cuda.synchronize()
    assert P.ops.device_error() == 0
