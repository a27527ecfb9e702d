"""The linear layer over 4-bit weights on the GPU against its 64-bit model (int4_model.linear)."""
import numpy as np
import pytest

import int4_model as model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def sp(lib_built):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import spmspm_b200
    spmspm_b200.reset_device_status()
    return spmspm_b200


def weight(rng, M, K, G):
    codes = rng.integers(0, 16, (M, K)).astype(np.uint8)
    scales = (rng.uniform(0.2, 1.0, (M, K // G)) * 0.01).astype(np.float16)
    zeros = rng.integers(0, 16, (M, K // G)).astype(np.uint8)
    return codes, scales, zeros


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def run(sp, rng, M, K, N, G, bias=False, relu=False, residual=False, x=None, W=None):
    codes, scales, zeros = weight(rng, M, K, G) if W is None else W
    x = rng.standard_normal((N, K)).astype(np.float16) if x is None else x
    b = rng.standard_normal(M).astype(np.float16) if bias else None
    r = rng.standard_normal((N, M)).astype(np.float16) if residual else None
    W = sp.pack_int4(dev(codes), dev(scales), dev(zeros))
    got = sp.linear_int4(W, dev(x), bias=dev(b) if bias else None, residual=dev(r) if residual else None,
                         activation=sp.ACT_RELU if relu else sp.ACT_NONE).cpu().numpy().astype(np.float64)
    f = lambda a: None if a is None else a.astype(np.float64)
    want, tol = model.linear(f(codes), f(scales), f(zeros), f(x), f(b), f(r), relu, fp16_weights=N > 16)
    err = np.abs(got - want)
    assert np.all(err <= tol), (float((err / tol).max()), np.argwhere(err > tol)[:4])
    assert sp.device_status() == 0
    return got


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("M,K", [(64, 128), (192, 384), (1024, 640), (64, 4096), (2368, 128)])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33])
def test_linear(sp, M, K, N, G):
    run(sp, np.random.default_rng(M + K + N + G), M, K, N, G)


@pytest.mark.parametrize("M,K,N,G", [(64, 64, 3, 64), (128, 192, 5, 32), (64, 320, 40, 64), (20480, 256, 8, 128), (20480, 256, 12, 64),
                                     (256, 16384, 1, 128), (320, 1024, 100, 128), (128, 64, 300, 32), (64, 128, 1000, 64), (448, 832, 129, 64)])
def test_linear_other_shapes(sp, M, K, N, G):
    run(sp, np.random.default_rng(M + K + N), M, K, N, G)


@pytest.mark.parametrize("N", [1, 13, 70])
@pytest.mark.parametrize("bias,relu,residual", [(True, False, False), (True, True, False), (False, True, True), (True, True, True)])
def test_tail(sp, N, bias, relu, residual):
    run(sp, np.random.default_rng(N), 320, 512, N, 64, bias, relu, residual)


def test_residual_may_be_the_output(sp):
    rng = np.random.default_rng(3)
    codes, scales, zeros = weight(rng, 128, 256, 128)
    W = sp.pack_int4(dev(codes), dev(scales), dev(zeros))
    for N in (3, 60):
        x, r = dev(rng.standard_normal((N, 256)).astype(np.float16)), dev(rng.standard_normal((N, 128)).astype(np.float16))
        want = sp.linear_int4(W, x, residual=r)
        assert torch.equal(sp.linear_int4(W, x, residual=r, out=r), want)


@pytest.mark.parametrize("N", [1, 64])
def test_special_values(sp, N):
    """Large and tiny x; a NaN in one row of x stays in its row; an infinite scale stays in its row of the weight."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((N, 256)).astype(np.float16)
    run(sp, rng, 128, 256, N, 64, x=(x * 1e4).clip(-60000, 60000).astype(np.float16))
    run(sp, rng, 128, 256, N, 64, x=(x * 1e-6).astype(np.float16))
    codes, scales, zeros = weight(rng, 128, 256, 64)
    scales[5, 1] = np.inf
    W = sp.pack_int4(dev(codes), dev(scales), dev(zeros))
    x[0, 3] = np.nan
    y = sp.linear_int4(W, dev(x)).cpu().numpy()
    bad = np.zeros(y.shape, bool)
    bad[0] = True
    bad[:, 5] = True
    assert not np.isfinite(y[bad]).any() and np.isfinite(y[~bad]).all()


@pytest.mark.parametrize("G", [32, 64, 128])
def test_decode_gives_the_weights(sp, G):
    rng = np.random.default_rng(5)
    codes, scales, zeros = weight(rng, 192, 384, G)
    W = sp.pack_int4(dev(codes), dev(scales), dev(zeros))
    s, z = np.repeat(scales.astype(np.float64), G, 1), np.repeat(zeros.astype(np.float64), G, 1)
    assert np.array_equal(sp.decode_int4(W).cpu().numpy(), (s * (codes - z)).astype(np.float16))


@pytest.mark.parametrize("G", [32, 64, 128])
def test_encode_is_the_nearest_code_and_keeps_zero(sp, G):
    rng = np.random.default_rng(6)
    A = (rng.standard_normal((128, 256)) * 0.02).astype(np.float16)
    A[rng.random(A.shape) < 0.3] = 0
    A[3, :G] = 0
    A[4, :G] = np.abs(A[4, :G]) + np.float16(0.01)
    A[5, 0] = 60000
    W = sp.encode_int4(dev(A), G)
    g = A.astype(np.float64).reshape(128, -1, G)
    lo, hi = np.minimum(g.min(-1, keepdims=True), 0), np.maximum(g.max(-1, keepdims=True), 0)
    s = ((hi - lo) / 15).astype(np.float16).astype(np.float64)
    back = sp.decode_int4(W).cpu().numpy().astype(np.float64).reshape(g.shape)
    # a code is off by half a step, the zero point by half a step more, the range by the rounding of s (15 codes of 2^-11)
    assert np.all(np.abs(back - g) <= s * (1 + 15 * 2.0 ** -11) + 2.0 ** -24)
    assert np.all(back[g == 0] == 0)


def test_graph_and_second_stream(sp):
    rng = np.random.default_rng(7)
    for N in (4, 96):
        codes, scales, zeros = weight(rng, 256, 512, 128)
        W = sp.pack_int4(dev(codes), dev(scales), dev(zeros))
        x = dev(rng.standard_normal((N, 512)).astype(np.float16))
        want = sp.linear_int4(W, x)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = sp.linear_int4(W, x)
        x2 = dev(rng.standard_normal((N, 512)).astype(np.float16))
        x.copy_(x2)
        graph.replay()
        assert torch.equal(y, sp.linear_int4(W, x2)) and not torch.equal(y, want)
