"""Calls on a stream given by hand (stream=): what they allocate must neither be memory that the current stream is still using nor go
back to the current stream while the given one is at work."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from spmspm_b200 import api  # noqa: E402


@pytest.fixture(scope="module")
def sp(lib_built):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import spmspm_b200
    spmspm_b200.reset_device_status()
    return spmspm_b200


def hold(stream=None, ms=30):
    """Keeps a stream busy for some milliseconds."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(ms * 2_000_000)


def half(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float16)).cuda()


def tensors(x):
    """The tensors a call has made."""
    if isinstance(x, torch.Tensor):
        return [x]
    return list(x) if isinstance(x, (tuple, list)) else [v for v in vars(x).values() if isinstance(v, torch.Tensor)]


def check(call):
    """call(stream) returns new tensors: the same bits with the given stream held up and the freed memory taken and filled at once, and
    with memory that the current stream still reads freed just before."""
    want = [t.clone() for t in tensors(call(None))]
    s = torch.cuda.Stream()
    call(s)                     # what a stream's first call prepares
    sizes = sorted({t.numel() * t.element_size() for t in want} | {1 << k for k in range(9, 23)})
    for side in ("given", "current"):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        if side == "given":     # the call's own temporaries come back while it has not even begun
            hold(s)
            got = call(s)
            others = [torch.full((n,), 0xA5, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
        else:                   # the current stream has freed memory that it has yet to read
            mine = [torch.full((n,), 0xA5, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
            s.wait_stream(torch.cuda.current_stream())
            hold()
            others = [t.clone() for t in mine]
            del mine
            got = call(s)
        s.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(tensors(got), want, strict=True))
        assert all(bool((t == 0xA5).all()) for t in others)
    if (0, s.cuda_stream) in api._initialised:
        api.release(s)


def test_preparing_four_bit_weights(sp):
    A = half(1, 512, 1024)
    check(lambda s: sp.encode_int4(A, 64, stream=s))
    rng = np.random.default_rng(2)
    codes, zeros = (torch.from_numpy(rng.integers(0, 16, (512, k)).astype(np.uint8)).cuda() for k in (1024, 16))
    scales = half(3, 512, 16).abs()
    check(lambda s: sp.pack_int4(codes, scales, zeros, stream=s))
    W = sp.encode_int4(A, 64)
    check(lambda s: sp.decode_int4(W, stream=s))


def test_bitmap_weights(sp):
    A, x, bias = half(4, 512, 1024) * (half(5, 512, 1024) > 0.4), half(6, 24, 1024), half(7, 512)
    check(lambda s: sp.encode_device(A, stream=s))
    W = sp.encode_device(A)
    for split_k in (1, 3):
        check(lambda s: sp.spmm(W, x, split_k=split_k, stream=s))
        check(lambda s: sp.linear(W, x, bias=bias, split_k=split_k, stream=s))
    Bc = sp.to_device(sp.init_sparse_matrix_a_bitmap_v6_b((half(8, 64, 1024) * (half(9, 64, 1024) > 0)).cpu().numpy()))
    check(lambda s: sp.decode_operand_b(Bc, stream=s))
    check(lambda s: sp.spmspm(W, Bc, split_k=2, stream=s))


@pytest.mark.parametrize("N", [3, 200])
@pytest.mark.parametrize("M,K", [(1024, 2048), (20480, 256)])
def test_linear(sp, M, K, N):
    W, x, bias = sp.encode_int4(half(10, M, K), 128), half(11, N, K), half(12, M)
    check(lambda s: sp.linear_int4(W, x, bias=bias, stream=s))


@pytest.mark.parametrize("T", [1, 96])
def test_cache(sp, T):
    """Appending with turned queries, reading and attention; T = 96 with the kernel for many rows."""
    B, L, heads, D = 3, 1000, 24, 64
    cache = sp.KvCacheInt4(B * 63, 16, heads, D)
    table = torch.arange(B * 63, dtype=torch.int32, device="cuda").view(B, 63)
    lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
    sp.kv_append(cache, half(13, B * L, heads, D), half(14, B * L, heads, D), table, lens)
    k, v, q = (half(i, B * T, heads, D) for i in (15, 16, 17))
    cos = torch.cos(torch.arange(L * 32, device="cuda").view(L, 32).float())
    sin = torch.sin(torch.arange(L * 32, device="cuda").view(L, 32).float())
    check(lambda s: sp.kv_append(cache, k, v, table, lens, q=q, cos=cos, sin=sin, stream=s))
    check(lambda s: sp.kv_read(cache, table, lens, n_tokens=B * T, stream=s))
    check(lambda s: sp.kv_attention(q, cache, table, lens, stream=s))
    assert sp.device_status() == 0


def test_a_stream_of_another_device_is_refused(sp):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    s = torch.cuda.Stream(device=1)
    A = half(1, 64, 128)
    W, cache = sp.encode_int4(A, 64), sp.KvCacheInt4(1, 16, 2, 64)
    table, lens, x = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), half(2, 1, 2, 64)
    for call in (lambda: sp.encode_int4(A, 64, stream=s), lambda: sp.linear_int4(W, half(3, 1, 128), stream=s),
                 lambda: sp.kv_append(cache, x, x, table, lens, stream=s), lambda: sp.kv_attention(x, cache, table, lens, stream=s)):
        with pytest.raises(sp.SpmmError, match="stream"):
            call()


def test_the_device_of_a_stream_is_looked_at(sp):
    """The check itself, against a device that is not the stream's."""
    s = torch.cuda.Stream()
    assert api._raw(s, torch.device("cuda", 0)) == s.cuda_stream and api._raw(None, "cpu") is None
    with pytest.raises(sp.SpmmError, match="stream"):
        api._raw(s, torch.device("cuda", 1))
    with pytest.raises(sp.SpmmError, match="stream"):
        api._on(torch.device("cuda", 1), s)


def captured(call, other):
    """What call() returns under a capture of the current stream; `other` is the stream it uses."""
    if (0, other.cuda_stream) in api._initialised:
        api.release(other)
    y = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
        y += 1
    assert (0, other.cuda_stream) not in api._initialised
    torch.cuda.synchronize()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((y == 1).all())
    return got, graph


@pytest.mark.parametrize("forked", [False, True])
def test_a_given_stream_while_the_current_one_is_captured(sp, forked):
    """A call beside the capture runs at once, one on a stream that is part of it is captured; neither ends it."""
    A, x = half(18, 256, 512), half(19, 8, 512)
    W, Q = sp.encode_device(A), sp.encode_int4(A, 128)
    want = sp.spmm(W, x, split_k=2), sp.linear_int4(Q, x)
    other = torch.cuda.Stream()

    def call():
        if forked:
            other.wait_stream(torch.cuda.current_stream())
        out = sp.spmm(W, x, split_k=2, stream=other), sp.linear_int4(Q, x, stream=other)
        if forked:
            torch.cuda.current_stream().wait_stream(other)
        return out

    got, graph = captured(call, other)
    # the schedule without scratch may add in another order: a last bit of each of two partial sums and of their sum
    assert bool(((got[0] - want[0]).abs() <= 3 * 2.0 ** -10 * want[0].abs().max()).all())
    assert torch.equal(got[1], want[1])
    if forked:
        x.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[1], -want[1])
