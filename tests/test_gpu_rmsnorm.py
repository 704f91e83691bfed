"""GPU: RMS norm + residual + int8 rows, bit for bit against a numpy restatement.

The sum of squares is taken in 64 bits on both sides, so the fp32 reciprocal root is the same number
and every step behind it is one named fp32 operation: tolerance 0.  (Two 64-bit sums in another order
differ by ~1e-16, so a different fp32 rounding of the root has a chance of about 1e-8 a row.)
"""
import ctypes as C

import numpy as np
import pytest
import torch

from fewbit_util import DT, int8_rows, ptr

pytestmark = pytest.mark.gpu


def restate(x, res, w, eps, name):
    """torch tensors on the CPU -> (sum or None, h fp32, aq, scale)."""
    dt = DT[name][1]
    s = x if res is None else (x.float() + res.float()).to(dt)
    v = s.float().numpy()
    ss = np.sum(v.astype(np.float64) ** 2, -1, keepdims=True)
    r = (1.0 / np.sqrt(ss / v.shape[-1] + float(np.float32(eps)))).astype(np.float32)
    h = (v * r).astype(np.float32)
    if w is not None:
        h = (h * w.numpy()).astype(np.float32)
    aq, sc = int8_rows(h)
    return (None if res is None else s), h, aq, sc


def run(sdq, x, res, w, eps, name, want_h=True, inplace=None, stream=None, ldx=0, ldr=0, M=None, K=None, flags=0):
    M, K = M or x.shape[0], K or x.shape[1]
    aq = torch.full((M, K), 77, dtype=torch.int8, device="cuda")
    sc = torch.full((M,), -1.0, device="cuda")
    h = torch.full((M, K), 5.0, dtype=x.dtype, device="cuda") if want_h else None
    out = None
    if res is not None:
        out = {None: None, "x": x, "residual": res}[inplace]
        if out is None:
            out = torch.zeros(M, K, dtype=x.dtype, device="cuda")
    lds = {None: 0, "x": ldx, "residual": ldr}[inplace]
    sdq.rmsnorm_quantize(ptr(x), DT[name][0], M, K, ptr(aq), ptr(sc), weight_ptr=ptr(w), eps=eps, residual_ptr=ptr(res),
                         sum_ptr=ptr(out), h_ptr=ptr(h), ldx=ldx, ldr=ldr, lds=lds, flags=flags, stream=stream)
    torch.cuda.synchronize()
    return out, h, aq, sc


def check(got, want, name):
    out, h, aq, sc = got
    s, hw, aqw, scw = want
    if s is not None:
        assert torch.equal(out.cpu().view(torch.uint8), s.contiguous().view(torch.uint8))
    assert np.array_equal(sc.cpu().numpy().view(np.uint32), scw.view(np.uint32))
    assert np.array_equal(aq.cpu().numpy(), aqw)
    if h is not None:
        hw, h = torch.from_numpy(hw).to(DT[name][1]), h.cpu()
        assert torch.equal(torch.isnan(h), torch.isnan(hw))
        assert torch.equal(torch.nan_to_num(h), torch.nan_to_num(hw))


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (1, 64), (5, 96), (2, 128), (7, 1000), (33, 264), (4, 1032), (2, 2048), (3, 4096),
                                 (1, 4104), (9, 5120), (2, 8192), (1, 14336), (2, 16384), (1, 16388), (1, 32768), (2, 33000), (300, 520)])
def test_bits(sdq, name, M, K):
    g = torch.Generator().manual_seed(M * 100003 + K)
    for with_res in (True, False):
        for with_w in (True, False):
            x = torch.randn(M, K, generator=g).to(DT[name][1])
            res = (3 * torch.randn(M, K, generator=g)).to(DT[name][1]) if with_res else None
            w = (1 + 0.3 * torch.randn(K, generator=g)) if with_w else None
            got = run(sdq, x.cuda(), None if res is None else res.cuda(), None if w is None else w.cuda(), 1e-6, name)
            check(got, restate(x, res, w, 1e-6, name), name)


def test_is_what_quantize_activations_makes_of_h(sdq):
    """To the last bit of a scale (one half step each for the multiplication and for the reciprocal of
    127, one for the division it stands for), and one code where that moves a value over a boundary."""
    x = torch.randn(50, 768, generator=torch.Generator().manual_seed(3))
    out, h, aq, sc = run(sdq, x.cuda(), None, None, 1e-5, "f32")
    aq2, sc2 = sdq.quantize_activations(h.cpu().numpy())
    assert (np.abs(sc.cpu().numpy() - sc2) <= 3 * 2.0 ** -24 * sc2).all()
    assert np.abs(aq.cpu().numpy().astype(int) - aq2).max() <= 1


@pytest.mark.parametrize("inplace", ["x", "residual"])
@pytest.mark.parametrize("name,K", [("bf16", 4096), ("f32", 515), ("f16", 40000)])
def test_in_place(sdq, inplace, name, K):
    g = torch.Generator().manual_seed(K)
    x, res = torch.randn(6, K, generator=g).to(DT[name][1]), torch.randn(6, K, generator=g).to(DT[name][1])
    got = run(sdq, x.cuda(), res.cuda(), None, 1e-6, name, inplace=inplace)
    check(got, restate(x, res, None, 1e-6, name), name)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("gap,shift", [(8, 0), (3, 0), (8, 1)])
def test_row_strides_and_alignment(sdq, name, gap, shift):
    """Rows that are slices of wider ones, and bases that are not 16-byte aligned."""
    M, K = 11, 640
    g = torch.Generator().manual_seed(gap)
    wide = torch.randn(M * (K + gap) + shift, generator=g).to(DT[name][1])
    res = torch.randn(M, K, generator=g).to(DT[name][1])
    x = torch.as_strided(wide, (M, K), (K + gap, 1), shift)
    d = wide.cuda()
    got = run(sdq, torch.as_strided(d, (M, K), (K + gap, 1), shift), res.cuda(), None, 1e-6, name, ldx=K + gap)
    check(got, restate(x.contiguous(), res, None, 1e-6, name), name)
    assert torch.equal(d.cpu(), wide)


def test_only_h_or_only_the_bytes(sdq):
    """A norm of queries asks for h alone; a norm in front of a linear for the bytes alone."""
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    _, h, aq, sc = restate(x, None, None, 1e-6, "bf16")
    d, got = x.cuda(), torch.empty(64, 128, dtype=torch.bfloat16, device="cuda")
    sdq.rmsnorm_quantize(ptr(d), 1, 64, 128, None, None, h_ptr=ptr(got), flags=0x10)
    assert torch.equal(got.cpu(), torch.from_numpy(h).bfloat16())
    check(run(sdq, d, None, None, 1e-6, "bf16", want_h=False), (None, h, aq, sc), "bf16")


def test_zero_rows_tiny_and_huge_values(sdq):
    x = torch.zeros(6, 512)
    x[1] = 1e-30
    x[2] = 1e18 * torch.randn(512, generator=torch.Generator().manual_seed(2))   # squares beyond fp32
    x[3, 5] = 3e38
    x[4] = 1e-42                                                                  # its reciprocal root is beyond fp32
    with np.errstate(all="ignore"):
        check(run(sdq, x.cuda(), None, None, 0.0, "f32"), restate(x, None, None, 0.0, "f32"), "f32")


def test_nan_stays_in_its_row(sdq):
    x = torch.randn(4, 1024, generator=torch.Generator().manual_seed(5))
    clean = run(sdq, x.cuda(), None, None, 1e-6, "f32")
    x[2, 100] = float("nan")
    got = run(sdq, x.cuda(), None, None, 1e-6, "f32")
    for i in (0, 1, 3):
        assert torch.equal(got[2][i], clean[2][i]) and torch.equal(got[3][i], clean[3][i])
    assert torch.isnan(got[1][2]).all()


def test_no_rows_and_no_columns(sdq):
    t = torch.full((4,), 9.0, device="cuda")
    sdq.rmsnorm_quantize(None, 0, 0, 64, None, None)
    sdq.rmsnorm_quantize(ptr(t), 0, 4, 0, ptr(t), ptr(t), flags=0x10)
    assert torch.equal(t.cpu(), torch.full((4,), 9.0))


def test_many_rows_and_another_stream(sdq):
    M, K = 20001, 256
    g = torch.Generator().manual_seed(9)
    x, res = torch.randn(M, K, generator=g).bfloat16(), torch.randn(M, K, generator=g).bfloat16()
    st = torch.cuda.Stream()
    dx, dr = x.cuda(), res.cuda()
    torch.cuda.synchronize()
    got = run(sdq, dx, dr, None, 1e-6, "bf16", stream=C.c_void_p(st.cuda_stream))
    check(got, restate(x, res, None, 1e-6, "bf16"), "bf16")
