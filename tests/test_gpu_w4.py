"""GPU: 4-bit weights -- the quantizer bit for bit, the products against 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from fewbit_util import DT, half_step, ptr

pytestmark = pytest.mark.gpu


def quantize_np(w, group, name):
    """numpy restatement of sdq_w4_quantize: (codes [N,K] in -7..7, scales [N,groups] as torch)."""
    N, K = w.shape
    groups = -(-K // group)
    pad = np.zeros((N, groups * group), np.float32)
    pad[:, :K] = w
    g = pad.reshape(N, groups, group)
    most = np.float32(torch.finfo(DT[name][1]).max)
    sc = torch.from_numpy(np.minimum(np.abs(g).max(-1) / np.float32(7), most)).to(DT[name][1])
    s = sc.float().numpy()[..., None]
    q = np.where(s > 0, np.clip(np.rint(g / np.where(s > 0, s, 1)), -7, 7), 0)
    return q.reshape(N, -1)[:, :K].astype(np.int8), sc


def pack_np(q):
    u = (q.astype(np.int32) + 8).astype(np.uint8)
    if u.shape[1] % 2:
        u = np.concatenate([u, np.full((u.shape[0], 1), 8, np.uint8)], 1)
    return u[:, 0::2] | (u[:, 1::2] << 4)


def full_range(rng, N, K, group, name):
    """Codes over the whole range -8..7 (other quantizers use -8) and positive scales."""
    q = rng.integers(-8, 8, (N, K)).astype(np.int8)
    sc = torch.from_numpy((0.001 + 0.01 * rng.random((N, -(-K // group)))).astype(np.float32)).to(DT[name][1])
    return q, sc


@pytest.mark.parametrize("src", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (3, 33, 32), (16, 64, 64), (17, 257, 128), (40, 1000, 64), (5, 130, 128)])
def test_quantizer_bits(sdq, src, scale, N, K, group):
    rng = np.random.default_rng(N * 1000 + K)
    w = torch.from_numpy((rng.standard_normal((N, K)) * 0.02).astype(np.float32)).to(DT[src][1])
    w[0] = 0
    if N > 2:
        w[2] *= 1e-3
    d = w.cuda()
    q = torch.full((N, (K + 1) // 2), 0xAA, dtype=torch.uint8, device="cuda")
    sc = torch.full((N, -(-K // group)), -1.0, device="cuda").to(DT[scale][1])
    sdq.w4_quantize(ptr(d), DT[src][0], N, K, group, ptr(q), ptr(sc), DT[scale][0], flags=0x10)
    qw, sw = quantize_np(w.float().numpy(), group, scale)
    assert torch.equal(sc.cpu().view(torch.uint8), sw.view(torch.uint8))
    assert np.array_equal(q.cpu().numpy(), pack_np(qw))


def test_quantizer_extreme_scales(sdq):
    """max|w| / 7 beyond fp16's largest number, and below its smallest."""
    w = torch.tensor([[6e5] + [1e5] * 31, [1e-9] * 32, [3e38] + [-1e38] * 31, [1e-40] * 32])
    d, q, sc = w.cuda(), torch.empty(4, 16, dtype=torch.uint8, device="cuda"), torch.empty(4, 1, dtype=torch.float16, device="cuda")
    sdq.w4_quantize(ptr(d), 0, 4, 32, 32, ptr(q), ptr(sc), 2, flags=0x10)
    qw, sw = quantize_np(w.numpy(), 32, "f16")
    assert torch.equal(sc.cpu(), sw) and np.array_equal(q.cpu().numpy(), pack_np(qw))


def gelu64(y):
    return 0.5 * y * (1 + np.tanh(np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3)))


def reference(x, xs, q, sc, group, bias, gelu):
    """(y, sum of |terms|) in 64 bits."""
    w = q.astype(np.float64) * np.repeat(sc.double().numpy(), group, 1)[:, :q.shape[1]]
    a = x * (1.0 if xs is None else xs.astype(np.float64)[:, None])
    y, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    return (gelu64(y) if gelu else y), mag


def tolerance(y, mag, K, group, out, gelu):
    """Every factor is exact or held in 22 bits (2^-22); products are added in fp32, at most 8 tensor
    steps inside a group (2^-23 each, the unit truncates), one fused multiply-add for each group and
    up to 16 partial sums (2^-24 each), and three more roundings for scale and bias -- all relative to
    the sum of the magnitudes.  GELU's slope stays below 1.13 and its exponential and division are
    good to 2^-20.  Then the output's rounding."""
    t = mag * (2.0 ** -22 + 8 * 2.0 ** -23 + (K / group + 16 + 3) * 2.0 ** -24)
    if gelu:
        t = 1.13 * t + 2.0 ** -20 * np.abs(y) + 2.0 ** -22
    tiny = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}[out]
    return t + half_step(out) * (np.abs(y) + t) + tiny


def activations(rng, M, K, name):
    a = (rng.standard_normal((M, K)) * np.exp(rng.normal(0, 1, (M, 1)))).astype(np.float32)
    if name == "i8":
        return torch.from_numpy(rng.integers(-127, 128, (M, K)).astype(np.int8)), (0.01 + rng.random(M)).astype(np.float32)
    return torch.from_numpy(a).to(DT[name][1]), None


def product(sdq, w, x, xs, M, N, out, bias=None, gelu=False, lda=0, stream=None, code=None):
    y = torch.full((M + 1, N), 3.0, device="cuda").to(DT[out][1])   # a row behind, to see it left alone
    dxs = None if xs is None else torch.from_numpy(xs).cuda()
    db = None if bias is None else torch.from_numpy(bias).cuda()
    sdq.w4_matmul(w, ptr(x), code if code is not None else {torch.int8: 3, torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype],
                  M, ptr(y), DT[out][0], a_scale_ptr=ptr(dxs), bias_ptr=ptr(db), gelu=gelu, lda=lda, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(y[M].float(), torch.full((N,), 3.0, device="cuda"))
    return y[:M].double().cpu().numpy()


def upload(sdq, q, sc, group, name):
    d, s = torch.from_numpy(pack_np(q)).cuda(), sc.cuda()
    return sdq.w4_upload(ptr(d), ptr(s), DT[name][0], q.shape[0], q.shape[1], group)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16", "i8"])
@pytest.mark.parametrize("group,scale", [(32, "f32"), (64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 64, 16), (1, 4096, 512), (2, 100, 33), (3, 1537, 70), (5, 256, 129), (7, 2048, 48),
                                   (8, 512, 1000), (9, 640, 17), (16, 1024, 64), (17, 333, 100), (24, 5000, 37), (33, 128, 40),
                                   (64, 700, 96), (65, 96, 24), (130, 160, 50)])
def test_products(sdq, kind, group, scale, M, K, N):
    rng = np.random.default_rng(M * 7919 + K * 31 + N)
    q, sc = full_range(rng, N, K, group, scale)
    w = upload(sdq, q, sc, group, scale)
    x, xs = activations(rng, M, K, kind)
    bias = rng.standard_normal(N).astype(np.float32)
    for out, b, gelu in (("f32", None, False), ("bf16", bias, False), ("f16", bias, True), ("f32", bias, True)):
        got = product(sdq, w, x.cuda(), xs, M, N, out, b, gelu)
        want, mag = reference(x.double().numpy(), xs, q, sc, group, b, gelu)
        tol = tolerance(want, mag, K, group, out, gelu)
        assert (np.abs(got - want) <= tol).all(), (out, np.max(np.abs(got - want) / tol))
    sdq.weight_release(w)


@pytest.mark.parametrize("M,K,N", [(1, 4096, 4096), (4, 14336, 1024), (20, 4096, 11008)])
def test_larger_products(sdq, M, K, N):
    rng = np.random.default_rng(K + N)
    q, sc = full_range(rng, N, K, 128, "bf16")
    w = upload(sdq, q, sc, 128, "bf16")
    for kind in ("bf16", "f32", "i8"):
        x, xs = activations(rng, M, K, kind)
        got = product(sdq, w, x.cuda(), xs, M, N, "f32")
        want, mag = reference(x.double().numpy(), xs, q, sc, 128, None, False)
        tol = tolerance(want, mag, K, 128, "f32", False)
        assert (np.abs(got - want) <= tol).all(), (kind, np.max(np.abs(got - want) / tol))
    sdq.weight_release(w)


def test_int8_rows_with_one_group_are_exact(sdq):
    """Integer sums below 2^24 and a scale of one: no rounding anywhere."""
    rng = np.random.default_rng(4)
    M, K, N = 6, 128, 200
    q = rng.integers(-8, 8, (N, K)).astype(np.int8)
    w = upload(sdq, q, torch.ones(N, 1), 128, "f32")
    x = rng.integers(-127, 128, (M, K)).astype(np.int8)
    got = product(sdq, w, torch.from_numpy(x).cuda(), np.ones(M, np.float32), M, N, "f32")
    assert np.array_equal(got, x.astype(np.int64) @ q.astype(np.int64).T)
    sdq.weight_release(w)


@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("gap,shift", [(16, 0), (1, 0), (16, 3)])
def test_row_strides_and_alignment(sdq, kind, gap, shift):
    rng = np.random.default_rng(gap + shift)
    M, K, N = 5, 320, 40
    q, sc = full_range(rng, N, K, 64, "f32")
    w = upload(sdq, q, sc, 64, "f32")
    x, xs = activations(rng, 1, M * (K + gap) + shift, kind)
    flat = x.flatten()
    view = torch.as_strided(flat, (M, K), (K + gap, 1), shift)
    xs = None if xs is None else np.repeat(xs, M)
    d = flat.cuda()
    got = product(sdq, w, torch.as_strided(d, (M, K), (K + gap, 1), shift), xs, M, N, "f32", lda=K + gap)
    want, mag = reference(view.double().numpy(), xs, q, sc, 64, None, False)
    assert (np.abs(got - want) <= tolerance(want, mag, K, 64, "f32", False)).all()
    sdq.weight_release(w)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_rows_stay_alone(sdq, kind, value):
    rng = np.random.default_rng(12)
    M, K, N = 10, 256, 48
    q, sc = full_range(rng, N, K, 64, "f32")
    q[:, 77] = np.where(q[:, 77] == 0, 3, q[:, 77])    # the poisoned column meets no zero
    w = upload(sdq, q, sc, 64, "f32")
    x, _ = activations(rng, M, K, kind)
    clean = product(sdq, w, x.cuda(), None, M, N, "f32")
    x[3, 77] = value
    got = product(sdq, w, x.cuda(), None, M, N, "f32")
    assert not np.isfinite(got[3]).any()
    if np.isinf(value):
        assert np.array_equal(got[3], value * np.sign(q[:, 77].astype(np.float64)))
    rest = np.arange(M) != 3
    assert np.array_equal(got[rest], clean[rest])
    sdq.weight_release(w)


def test_magnitudes_do_not_matter(sdq):
    """Rows from 1e-38 to 1e30: every row keeps fp32's relative precision."""
    rng = np.random.default_rng(13)
    M, K, N = 8, 512, 32
    q, sc = full_range(rng, N, K, 128, "f32")
    w = upload(sdq, q, sc, 128, "f32")
    x = (rng.standard_normal((M, K)) * np.array([1e-38, 1e-30, 1e-10, 1e-4, 1.0, 1e5, 1e20, 1e30])[:, None]).astype(np.float32)
    got = product(sdq, w, torch.from_numpy(x).cuda(), None, M, N, "f32")
    want, mag = reference(x.astype(np.float64), None, q, sc, 128, None, False)
    tol = tolerance(want, mag, K, 128, "f32", False)
    tol[0] += 2.0 ** -149 * K          # products of subnormal size round to the subnormal grid
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol, 1)
    sdq.weight_release(w)


def test_host_upload_lookup_and_wrong_handles(sdq, pkg):
    rng = np.random.default_rng(2)
    q, sc = full_range(rng, 24, 96, 32, "f16")
    packed, scale = pack_np(q), np.ascontiguousarray(sc.numpy())
    h = sdq.w4_upload(packed.ctypes.data, scale.ctypes.data, 2, 24, 96, 32, flags=pkg.sdq.SRC_HOST)
    assert sdq.weight_lookup(packed.ctypes.data) == h
    assert sdq.weight_info(h)[:2] == (24, 96) and sdq.weight_info(h)[2] is None
    x, _ = activations(rng, 2, 96, "f32")
    got = product(sdq, h, x.cuda(), None, 2, 24, "f32")
    want, mag = reference(x.double().numpy(), None, q, sc, 32, None, False)
    assert (np.abs(got - want) <= tolerance(want, mag, 96, 32, "f32", False)).all()
    d = x.cuda()
    for call in (lambda: sdq.qgemm(h, ptr(d), 2, ptr(d)), lambda: sdq.w4_matmul(h + 999, ptr(d), 0, 2, ptr(d))):
        with pytest.raises(pkg.SdqError) as e:
            call()
        assert e.value.code == 1 and "handle" in e.value.msg
    w8 = sdq.weight_upload(np.ones((8, 96), np.int8), np.ones(8, np.float32))
    with pytest.raises(pkg.SdqError) as e:
        sdq.w4_matmul(w8, ptr(d), 0, 2, ptr(d))
    assert "not a 4-bit weight" in e.value.msg
    with pytest.raises(pkg.SdqError) as e:
        sdq.w4_matmul(h, ptr(d), 0, 2, ptr(d), lda=95)
    assert "stride" in e.value.msg
    sdq.weight_release(h)
    with pytest.raises(pkg.SdqError):
        sdq.w4_matmul(h, ptr(d), 0, 2, ptr(d))
    sdq.weight_release(w8)


def test_no_rows(sdq):
    rng = np.random.default_rng(2)
    q, sc = full_range(rng, 8, 32, 32, "f32")
    w = upload(sdq, q, sc, 32, "f32")
    sdq.w4_matmul(w, None, 0, 0, None)
    sdq.weight_release(w)


def test_replayed_from_a_graph_and_on_two_streams(sdq):
    """Two graphs captured on one stream and replayed side by side: the calls share no scratch."""
    rng = np.random.default_rng(21)
    M, K, N = 4, 4096, 1024
    q, sc = full_range(rng, N, K, 128, "bf16")
    w = upload(sdq, q, sc, 128, "bf16")
    xs = [activations(rng, M, K, "bf16")[0].cuda() for _ in range(2)]
    want = [product(sdq, w, x, None, M, N, "f32") for x in xs]
    ys = [torch.zeros(M, N, device="cuda") for _ in range(2)]
    st, graphs = torch.cuda.Stream(), []
    for x, y in zip(xs, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(3):
                sdq.w4_matmul(w, ptr(x), 1, M, ptr(y), stream=C.c_void_p(st.cuda_stream))
        graphs.append(g)
    sts = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, s in zip(graphs, sts):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for y, t in zip(ys, want):
        assert np.array_equal(y.double().cpu().numpy(), t)
    sdq.weight_release(w)
