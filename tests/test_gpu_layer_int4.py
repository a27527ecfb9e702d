"""The 4-bit operators together, as a decoder layer runs them: 4-bit weights, append to the paged cache, attention over it.  Every step
is checked on the tensors the step before really produced, so that a rounding upstream cannot hide or fake an error."""
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


def f64(t):
    return t.cpu().numpy().astype(np.float64)


class Taps:
    """Records the inputs and outputs of a layer's steps."""

    def __init__(self, layer):
        self.linear, self.attend = [], []
        run_linear, run_attend = layer._linear, layer._attend

        def linear(name, x, bias=None, residual=None, relu=False):
            y = run_linear(name, x, bias, residual, relu)
            self.linear.append((name, x.clone(), bias, None if residual is None else residual.clone(), relu, y.clone()))
            return y

        def attend(qkv, T):
            y = run_attend(qkv, T)
            self.attend.append((qkv.clone(), T, y.clone()))
            return y
        layer._linear, layer._attend = linear, attend


@pytest.mark.parametrize("hidden,heads,page", [(256, 4, 16), (512, 4, 64)])
@pytest.mark.parametrize("T", [5, 70])
def test_layer_steps(sp, hidden, heads, page, T):
    from spmspm_b200.layer import SparseOptDecoderLayer, _gen
    dev = torch.device("cuda", 0)
    B, d = 2, hidden // heads
    layer = SparseOptDecoderLayer(hidden, heads, 4 * hidden, 0.0, dev, batch=B, max_len=T + 8, keep_dense=True, weights="int4", kv_cache="int4",
                                  page_size=page)
    taps = Taps(layer)
    layer.reset()
    layer.forward(_gen((B * T, hidden), 3, dev, 1.0), T)
    for i in range(3):
        layer.forward(_gen((B, hidden), 4 + i, dev, 1.0), 1)
    assert layer.kv_lens.tolist() == [T + 3] * B and int(layer.pos.item()) == T + 3
    for name, x, bias, residual, relu, y in taps.linear:
        # the decoded weight is s (c - z) rounded to fp16: 2^-11 of itself away from the unrounded one that few rows are multiplied with
        W, N = f64(layer.dense[name]), x.shape[0]
        xx = f64(x)
        want = xx @ W.T
        mag = np.abs(xx) @ np.abs(W).T
        # fp32 sums: K / 16 + 64 additions of terms s c |x| and s z |x|, which are at most 15 s |x| each, and s <= 2 max |w| / 15
        peak = np.repeat(np.abs(W).reshape(W.shape[0], -1, layer.W[name].group).max(-1), layer.W[name].group, 1)
        tol = 2.0 ** -11 * mag + (W.shape[1] / 16 + 64) * 2.0 ** -24 * 4 * (np.abs(xx) @ peak.T)
        want = want + f64(bias)
        want = np.maximum(want, 0) if relu else want
        want = want + f64(residual) if residual is not None else want
        assert np.all(np.abs(f64(y) - want) <= tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -24), name
    seen = [(np.zeros((0, heads, d)), np.zeros((0, heads, d))) for _ in range(B)]
    for qkv, t, y in taps.attend:
        q, k, v = (f64(x).reshape(B, t, heads, d) for x in qkv.split(hidden, dim=1))
        for b in range(B):
            seen[b] = tuple(np.concatenate([old, new[b]]) for old, new in zip(seen[b], (k, v)))
            kk, vv, sc = model.entry(seen[b][0]), model.entry(seen[b][1]), model.scaled_codes(seen[b][1])
            want, tol = model.attention(q[b], kk, vv, sc, d ** -0.5)
            assert np.all(np.abs(f64(y).reshape(B, t, heads, d)[b] - want) <= tol)
    assert sp.device_status() == 0


def test_four_bit_cache_stays_near_the_dense_one(sp):
    """The same layer with either cache.  Keys and values are held within s / 2, where s <= (max - min) / 15 of their 32 channels (1 % for
    the roundings of s, m and the divisions).  A score moves by at most delta = |q|_1 s_k / 2 / sqrt(d), a softmax weight by a factor within
    exp(2 delta), the output by s_v / 2 + (exp(2 delta) - 1) max |v|; 2^-8 max |v| is for the fp16 of both paths."""
    from spmspm_b200.layer import SparseOptDecoderLayer, _gen
    dev = torch.device("cuda", 0)
    kw = dict(batch=2, max_len=40, keep_dense=True)
    outs = []
    for cache in ("dense", "int4"):
        layer = SparseOptDecoderLayer(256, 4, 1024, 0.6, dev, kv_cache=cache, **kw)
        taps = Taps(layer)
        layer.forward(_gen((2 * 32, 256), 3, dev, 1.0), 32)
        outs.append(taps.attend[0])
    assert torch.equal(outs[0][0], outs[1][0])
    q, k, v = (f64(t).reshape(-1, 2, 32) for t in outs[0][0].split(256, dim=1))
    step_k, step_v = ((t.max(-1) - t.min(-1)).max() / 15 * 1.01 for t in (k, v))
    delta = np.abs(q).sum((-1, -2)).max() * step_k / 2 / 8
    bound = step_v / 2 + (np.exp(2 * delta) - 1 + 2.0 ** -8) * np.abs(v).max()
    diff = np.abs(f64(outs[0][2]) - f64(outs[1][2]))
    assert 0 < diff.max() <= bound


def test_generation_with_four_bit_weights_and_cache(sp):
    from spmspm_b200.layer import SparseOptDecoderLayer, generate_timed
    dev = torch.device("cuda", 0)
    layer = SparseOptDecoderLayer(256, 4, 1024, 0.0, dev, batch=2, max_len=24, weights="int4", kv_cache="int4", page_size=16)
    for use_graph in (False, True):
        total, pre, per_step, graphed = generate_timed(layer, 8, 12, steps=1, warmup=1, use_graph=use_graph)
        assert total > 0 and pre > 0 and per_step > 0 and (graphed or not use_graph)
        assert int(layer.pos.item()) == 20 and layer.kv_lens.tolist() == [20, 20]
    assert sp.device_status() == 0


def test_module_and_operator(sp):
    """Int4Linear / torch.ops.spmspm_b200.int4_linear: the bits of linear_int4, shapes under a fake tensor, any leading dimensions."""
    from spmspm_b200.ops import Int4Linear
    torch.manual_seed(0)
    W = sp.encode_int4((torch.randn(192, 128, device="cuda") * 0.02).half(), 64)
    bias = torch.randn(192, device="cuda").half()
    lin = Int4Linear(W, bias, activation=sp.ACT_RELU)
    x, r = torch.randn(3, 5, 128, device="cuda").half(), torch.randn(3, 5, 192, device="cuda").half()
    want = sp.linear_int4(W, x.reshape(15, 128), bias=bias, residual=r.reshape(15, 192), activation=sp.ACT_RELU)
    assert torch.equal(lin(x, r).reshape(15, 192), want)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        y = torch.ops.spmspm_b200.int4_linear(mode.from_tensor(x)[0], mode.from_tensor(W.data), 192, 64, None, None, 0)
    assert tuple(y.shape) == (5, 192) and y.dtype == torch.float16


def test_layer_refuses(lib_built):
    from spmspm_b200.layer import SparseOptDecoderLayer
    for bad in (dict(weights="int8"), dict(kv_cache="fp8")):
        with pytest.raises(ValueError):
            SparseOptDecoderLayer(256, 4, 1024, 0.0, torch.device("cuda", 0), batch=1, max_len=8, **bad)


FIRST_CALLS_CAPTURED = """
import torch, spmspm_b200 as sp
torch.manual_seed(0)
x = torch.randn(4, 256, device="cuda").half()
codes = torch.randint(0, 16, (768, 256), device="cuda", dtype=torch.uint8)
scales, zeros = torch.full((768, 2), 0.01, device="cuda").half(), torch.full((768, 2), 8, device="cuda", dtype=torch.uint8)
W = sp.pack_int4(codes, scales, zeros)
cache = sp.KvCacheInt4(8, 16, 2, 128)
table, lens = torch.arange(8, device="cuda", dtype=torch.int32).view(4, 2), torch.full((4,), 1, device="cuda", dtype=torch.int32)

def step():
    q, k, v = (t.unflatten(1, (2, 128)) for t in sp.linear_int4(W, x).split(256, dim=1))
    sp.kv_append(cache, k, v, table, lens)
    return sp.kv_attention(q, cache, table, lens)

torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = step()
g.replay()
torch.cuda.synchronize()
first = y.clone()
assert torch.equal(step(), first) and bool(first.any()) and sp.device_status() == 0
print("same")
"""


def test_first_calls_of_a_process_may_be_captured(lib_built):
    import subprocess
    import sys
    got = subprocess.run([sys.executable, "-c", FIRST_CALLS_CAPTURED], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "same", got.stderr[-2000:]


def test_broadcast_keys_and_queries(sp):
    """Strides of zero: one key and value for all heads, one query for all tokens."""
    torch.manual_seed(1)
    B, H, D = 3, 4, 64
    table, lens = torch.arange(6, device="cuda", dtype=torch.int32).view(B, 2), torch.full((B,), 1, device="cuda", dtype=torch.int32)
    k, v, q = (torch.randn(*s, device="cuda").half() for s in ((B, 1, D), (B, 1, D), (1, H, D)))
    outs = []
    for dense in (False, True):
        kk, vv, qq = k.expand(B, H, D), v.expand(B, H, D), q.expand(B, H, D)
        if dense:
            kk, vv, qq = kk.contiguous(), vv.contiguous(), qq.contiguous()
        cache = sp.KvCacheInt4(6, 16, H, D)
        sp.kv_append(cache, kk, vv, table, lens)
        outs.append((cache.pool.clone(), sp.kv_attention(qq, cache, table, lens)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert sp.device_status() == 0


def test_steps_on_two_streams_at_once(sp):
    """Two users with caches, tensors and streams of their own, steps interleaved: the bits of one after the other."""
    torch.manual_seed(2)
    B, H, D, steps = 5, 8, 128, 6
    W = sp.encode_int4((torch.randn(3 * H * D, H * D, device="cuda") * 0.02).half())

    def user(seed, stream):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = [torch.randn(B, H * D, device="cuda", generator=g).half() for _ in range(steps)]
        cache = sp.KvCacheInt4(B * 4, 16, H, D)
        table, lens = torch.arange(B * 4, device="cuda", dtype=torch.int32).view(B, 4), torch.zeros(B, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()

        def step(i):
            with torch.cuda.stream(stream):
                q, k, v = (t.unflatten(1, (H, D)) for t in sp.linear_int4(W, x[i]).split(H * D, dim=1))
                lens.add_(1)
                sp.kv_append(cache, k, v, table, lens)
                return sp.kv_attention(q, cache, table, lens)
        return step
    alone = []
    for seed in (1, 2):
        step = user(seed, torch.cuda.current_stream())
        alone.append([step(i) for i in range(steps)])
    a, b = user(1, torch.cuda.Stream()), user(2, torch.cuda.Stream())
    both = [(a(i), b(i)) for i in range(steps)]
    torch.cuda.synchronize()
    for i, (x, y) in enumerate(both):
        assert torch.equal(x, alone[0][i]) and torch.equal(y, alone[1][i])
    assert sp.device_status() == 0
