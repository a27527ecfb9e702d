"""The paged 4-bit key/value cache on the GPU against the 64-bit models of int4_model.py: what is written has to be there bit for
bit; attention has to stay within the error that its roundings allow."""
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


def f16(rng, *shape, scale=1.0):
    x = rng.standard_normal(shape) * scale
    if len(shape) > 1:
        x = x + 2 * rng.standard_normal(shape[-2:]) * (rng.random(shape[-2:]) < 0.1)
    return x.astype(np.float16)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Batch:
    """Sequences of given lengths on shuffled pages; the last q_lens[b] tokens of each are new."""

    def __init__(self, sp, rng, lens, q_lens, heads, D, page, spare=2):
        self.sp, self.lens, self.q_lens, self.heads, self.D, self.page = sp, list(lens), list(q_lens), heads, D, page
        per = [-(-n // page) for n in lens]
        total = sum(per) + spare
        order = rng.permutation(total).astype(np.int32)
        table = np.full((len(lens), max(max(per), 1)), -1, np.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_h, self.spare_pages = table, order[at:]
        self.cache = sp.KvCacheInt4(total, page, heads, D)
        self.table, self.kv_lens = dev(table), i32(lens)
        self.cu = i32(np.concatenate([[0], np.cumsum(q_lens)]))
        self.full_cu = i32(np.concatenate([[0], np.cumsum(lens)]))
        self.k = [f16(rng, n, heads, D) for n in lens]
        self.v = [f16(rng, n, heads, D) for n in lens]

    def fill(self):
        k, v = (np.concatenate(x) if sum(self.lens) else np.zeros((0, self.heads, self.D), np.float16) for x in (self.k, self.v))
        self.sp.kv_append(self.cache, dev(k), dev(v), self.table, self.kv_lens, cu_q=self.full_cu)
        return self

    def held(self, b):
        v = self.v[b].astype(np.float64)
        return model.entry(self.k[b].astype(np.float64)), model.entry(v), model.scaled_codes(v)


def is_tall(bt, Hq, t):
    """Whether a sequence with t new tokens goes to the kernel for many rows, which takes keys and values as kv_read returns them."""
    group = Hq // bt.heads
    return (max(bt.q_lens) * group >= 64 and -(-sum(bt.q_lens) * group // 256) * bt.heads >= 24 and t * group >= 64)


def reference(bt, b, q, Hq, scale, tweak=None):
    k, v, sc = bt.held(b)
    if is_tall(bt, Hq, bt.q_lens[b]):
        with np.errstate(over="ignore"):
            k, v, sc = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64), 0 * sc
    if tweak is not None:
        tweak(k, v, sc)
    return model.attention(q.astype(np.float64), k, v, sc, scale)


def check_attention(sp, rng, bt, Hq, scale=None, uniform=False, q=None, **kw):
    n = sum(bt.q_lens)
    q = f16(rng, n, Hq, bt.D) if q is None else q
    out = torch.full((n, Hq, bt.D), 7.0, dtype=torch.float16, device="cuda")
    got = sp.kv_attention(dev(q), bt.cache, bt.table, bt.kv_lens, cu_q=None if uniform else bt.cu, max_q=max(bt.q_lens), scale=scale, out=out, **kw)
    got = got.cpu().numpy().astype(np.float64)
    at = 0
    for b, t in enumerate(bt.q_lens):
        want, tol = reference(bt, b, q[at:at + t], Hq, bt.D ** -0.5 if scale is None else scale)
        err = np.abs(got[at:at + t] - want)
        assert np.all(err <= tol), (b, t, bt.lens[b], float((err - tol).max()), float((err / np.maximum(tol, 1e-30)).max()))
        at += t
    assert sp.device_status() == 0


# ------------------------------------------------------------------------------------------------ append and read

@pytest.mark.parametrize("D,heads,page", [(128, 1, 16), (128, 5, 64), (64, 3, 32), (64, 8, 128), (128, 8, 48)])
@pytest.mark.parametrize("lens,q_lens", [((1,), (1,)), ((17, 16, 15), (17, 16, 15)), ((33, 1, 70, 200), (1, 1, 5, 131)), ((9, 40), (0, 3))])
def test_what_is_appended_is_held_bit_for_bit(sp, D, heads, page, lens, q_lens):
    rng = np.random.default_rng(D + heads + page + sum(lens))
    bt = Batch(sp, rng, lens, q_lens, heads, D, page)
    new = [np.concatenate([x[b][n - t:] for b, (n, t) in enumerate(zip(lens, q_lens))]) for x in (bt.k, bt.v)]
    sp.kv_append(bt.cache, dev(new[0]), dev(new[1]), bt.table, bt.kv_lens, cu_q=bt.cu)
    k, v = sp.kv_read(bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, n_tokens=sum(q_lens))
    for got, want in ((k, new[0]), (v, new[1])):
        assert np.array_equal(got.cpu().numpy(), model.entry(want.astype(np.float64)).astype(np.float16))
    assert sp.device_status() == 0


@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (128, 64, True), (64, 64, True), (64, 8, False), (128, 24, False), (128, 40, True)])
def test_rotation_is_rounded_once(sp, D, rot, interleaved):
    rng = np.random.default_rng(rot)
    lens, q_lens, heads, Hq = (300, 5, 2049), (40, 5, 1), 3, 6
    bt = Batch(sp, rng, lens, q_lens, heads, D, 32)
    n = sum(q_lens)
    ang = np.arange(2049)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    k, v, q = f16(rng, n, heads, D), f16(rng, n, heads, D), f16(rng, n, Hq, D)
    pos = np.concatenate([np.arange(a - b, a) for a, b in zip(lens, q_lens)])
    got_q = sp.kv_append(bt.cache, dev(k), dev(v), bt.table, bt.kv_lens, cu_q=bt.cu, q=dev(q), cos=dev(cos), sin=dev(sin), interleaved=interleaved)
    want_q = model.rotate(q.astype(np.float64), pos, cos, sin, interleaved)
    assert np.array_equal(got_q.cpu().numpy(), want_q.astype(np.float16))
    gk, gv = sp.kv_read(bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, n_tokens=n)
    assert np.array_equal(gk.cpu().numpy(), model.entry(model.rotate(k.astype(np.float64), pos, cos, sin, interleaved)).astype(np.float16))
    assert np.array_equal(gv.cpu().numpy(), model.entry(v.astype(np.float64)).astype(np.float16))


def test_extreme_groups(sp):
    """Constant groups, the largest finite values, subnormals, signed zeros, infinities and NaN."""
    D, heads = 128, 2
    x = np.zeros((6, heads, D), np.float16)
    x[0, :, :32] = 3.25
    x[1, :, :32] = np.linspace(-65504, 65504, 32)
    x[1, :, 32:64] = 65504
    x[2, :, :32] = np.arange(32) * 6e-8
    x[2, :, 32:64] = np.where(np.arange(32) % 2, -0.0, 0.0)
    x[3, 0, 5] = np.inf
    x[3, 1, 40] = np.nan
    x[4, :, 64:96] = np.where(np.arange(32) % 2, 1e-3, 60000)
    x[5] = np.random.default_rng(0).standard_normal((heads, D)) * 1e4
    bt = Batch(sp, np.random.default_rng(1), (6,), (6,), heads, D, 16)
    sp.kv_append(bt.cache, dev(x), dev(x), bt.table, bt.kv_lens)
    want = model.entry(x.astype(np.float64)).astype(np.float16)
    for got in sp.kv_read(bt.cache, bt.table, bt.kv_lens, n_tokens=6):
        got = got.cpu().numpy()
        assert np.array_equal(got, want, equal_nan=True)
        assert np.isnan(got[3, 0, :32]).all() and np.isfinite(got[3, 0, 32:]).all()


def test_append_takes_strided_views_and_leaves_the_rest_alone(sp):
    """k, v and q as slices of one fused projection; rows behind the last sequence and pages of others stay as they were."""
    rng = np.random.default_rng(5)
    D, heads, Hq, n = 64, 2, 4, 9
    bt = Batch(sp, rng, (20, 4), (5, 2), heads, D, 16)
    fused = dev(f16(rng, n, Hq + 2 * heads, D))
    q, k, v = fused[:, :Hq], fused[:, Hq:Hq + heads], fused[:, Hq + heads:]
    bt.cache.pool.fill_(0xA5)
    before = bt.cache.pool.clone()
    cos = torch.ones((64, D // 2), device="cuda")
    q_out = torch.full((n, Hq, D), 7.0, dtype=torch.float16, device="cuda")
    sp.kv_append(bt.cache, k, v, bt.table, bt.kv_lens, cu_q=bt.cu, q=q, cos=cos, sin=torch.zeros_like(cos), q_out=q_out)
    assert torch.equal(q_out[:7], q[:7]) and bool((q_out[7:] == 7).all())
    gk, gv = sp.kv_read(bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, n_tokens=7)
    assert np.array_equal(gk.cpu().numpy(), model.entry(k[:7].cpu().numpy().astype(np.float64)).astype(np.float16))
    assert np.array_equal(gv.cpu().numpy(), model.entry(v[:7].cpu().numpy().astype(np.float64)).astype(np.float16))
    changed = (bt.cache.pool != before).view(-1, heads, 20 * D)          # [page, head, bytes] (pages of one block)
    assert changed.shape[0] == bt.cache.num_pages
    touched = {int(bt.table_h[0, 0]), int(bt.table_h[0, 1]), int(bt.table_h[1, 0])}
    for p in range(bt.cache.num_pages):
        assert bool(changed[p].any()) == (p in touched)
    # tokens 0..14 of the first sequence's first page were not new: at most one token's worth of its bytes changed
    assert int(changed[int(bt.table_h[0, 0])].sum()) <= heads * 2 * (D // 2 + D // 8)


def test_bad_pages_and_positions_are_reported_and_skipped(sp):
    """A page number outside the pool, a token past the table and one past the angles set the status word and touch nothing; rows
    before the start of the context are skipped silently."""
    rng = np.random.default_rng(6)
    D, heads = 64, 2
    x = dev(f16(rng, 4, heads, D))
    cache = sp.KvCacheInt4(3, 16, heads, D)
    for table, lens, angles in (([[5]], [4], 0), ([[-1]], [4], 0), ([[1]], [20], 0), ([[1]], [4], 2)):
        cache.pool.fill_(0xA5)
        sp.reset_device_status()
        table, lens = torch.tensor(table, dtype=torch.int32, device="cuda"), i32(lens)
        cos = torch.ones((angles, 4), device="cuda") if angles else None
        sp.kv_append(cache, x, x, table, lens, cos=cos, sin=cos)
        assert sp.device_status() == 8
        if not angles:
            assert bool((cache.pool == 0xA5).all())
            sp.reset_device_status()
            k, v = sp.kv_read(cache, table, lens, n_tokens=4)
            assert sp.device_status() == 8 and not bool(k.any()) and not bool(v.any())
            sp.reset_device_status()
            o = sp.kv_attention(x, cache, table, lens)
            assert sp.device_status() == 8
            if int(lens[0]) <= 16:
                assert not bool(o.any())
    sp.reset_device_status()
    cache.pool.fill_(0xA5)
    sp.kv_append(cache, x, x, torch.tensor([[1]], dtype=torch.int32, device="cuda"), i32([0]))
    assert sp.device_status() == 0 and bool((cache.pool == 0xA5).all())


# ------------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("D,Hkv,group,page", [(128, 2, 1, 64), (128, 2, 8, 16), (64, 3, 4, 32), (128, 1, 16, 128), (64, 2, 20, 48), (128, 1, 7, 16)])
@pytest.mark.parametrize("lens", [(1,), (2, 16, 17), (63, 64, 65, 129), (1000, 3)])
def test_single_token_attention(sp, D, Hkv, group, page, lens):
    rng = np.random.default_rng(D + group + sum(lens))
    bt = Batch(sp, rng, lens, [1] * len(lens), Hkv, D, page).fill()
    check_attention(sp, rng, bt, Hkv * group, uniform=True)


@pytest.mark.parametrize("D,Hkv,group", [(128, 2, 1), (64, 2, 4), (128, 1, 8)])
@pytest.mark.parametrize("lens,q_lens", [((5,), (5,)), ((100, 64, 200), (3, 1, 8)), ((130, 20, 77), (130, 0, 33)), ((40, 300), (17, 100))])
def test_several_new_tokens_are_causal(sp, D, Hkv, group, lens, q_lens):
    rng = np.random.default_rng(D + group + sum(lens))
    bt = Batch(sp, rng, lens, q_lens, Hkv, D, 32).fill()
    check_attention(sp, rng, bt, Hkv * group)


@pytest.mark.parametrize("D,Hkv,group", [(128, 24, 1), (64, 24, 1), (128, 8, 8), (64, 8, 5), (128, 24, 2)])
@pytest.mark.parametrize("lens,q_lens", [((128,), (128,)), ((300, 70, 513), (299, 64, 129)), ((257, 40, 9, 700), (256, 3, 0, 65)), ((1000, 90), (130, 90))])
def test_many_new_tokens(sp, D, Hkv, group, lens, q_lens):
    """Prompts and chunks, with short sequences among them: row tiles that end inside, that see nothing of a key tile, odd groups."""
    rng = np.random.default_rng(D + group + sum(lens))
    bt = Batch(sp, rng, lens, q_lens, Hkv, D, 16 if D == 64 else 64).fill()
    assert any(is_tall(bt, Hkv * group, t) for t in q_lens)
    check_attention(sp, rng, bt, Hkv * group)


def test_many_new_tokens_uniform_and_without_a_bound(sp):
    rng = np.random.default_rng(21)
    bt = Batch(sp, rng, (150, 140), (140, 140), 24, 64, 32).fill()
    check_attention(sp, rng, bt, 24, uniform=True)
    q = dev(f16(rng, 280, 24, 64))
    want = sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens)
    assert torch.equal(sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu), want)
    assert torch.equal(sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens, max_q=280), want)


@pytest.mark.parametrize("D", [64, 128])
def test_many_new_tokens_with_nothing_to_see_and_nan(sp, D):
    """More new tokens than the cache holds; NaN behind the context, and in values and keys that only some rows may see."""
    rng = np.random.default_rng(22)
    bt = Batch(sp, rng, (150, 400, 0), (200, 300, 70), 24, D, 64)
    bt.cache.pool.view(torch.float16).fill_(float("nan"))
    bt.k[0], bt.v[0] = bt.k[0][:150], bt.v[0][:150]
    bt.v[1][230, 3, 40] = np.nan       # rows 130.. of the second sequence see token 230
    bt.k[1][399, 5, 3] = np.inf        # its last row alone sees token 399
    bt.fill()
    q = f16(rng, 570, 24, D)
    out = sp.kv_attention(dev(q), bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, max_q=300).cpu().numpy().astype(np.float64)
    assert not out[:50].any() and not out[500:].any()
    want, tol = reference(bt, 0, q[50:200], 24, D ** -0.5)
    assert np.all(np.abs(out[50:200] - want) <= tol)

    def tweak(k, v, sc):
        v[np.isnan(v)] = 0
        k[np.isnan(k)] = 0
        sc[np.isnan(sc)] = 0
    want, tol = reference(bt, 1, q[200:500], 24, D ** -0.5, tweak)
    got = out[200:500]
    bad = np.zeros(got.shape, bool)
    bad[130:, 3, 32:64] = True
    bad[299, 5] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad])
    assert sp.device_status() == 0


def test_many_new_tokens_bad_pages(sp):
    """A page number outside the pool: its tokens count as unseen, the rest as if they were all there is."""
    rng = np.random.default_rng(23)
    bt = Batch(sp, rng, (320,), (100,), 24, 64, 64).fill()
    q = f16(rng, 100, 24, 64)
    table = bt.table_h.copy()
    table[0, 1] = 1000
    sp.reset_device_status()
    out = sp.kv_attention(dev(q), bt.cache, dev(table), bt.kv_lens, max_q=100).cpu().numpy().astype(np.float64)
    assert sp.device_status() == 8
    sp.reset_device_status()
    k, v, sc = bt.held(0)
    keep = np.r_[0:64, 128:320]
    want, tol = model.attention(q.astype(np.float64), k[keep].astype(np.float16).astype(np.float64), v[keep].astype(np.float16).astype(np.float64),
                                0 * sc[keep], 0.125)
    assert np.all(np.abs(out - want) <= tol)


def test_many_sequences_and_empty_ones(sp):
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(1, 90, 150)]
    q_lens = [int(x) for x in rng.integers(0, 3, 150)]
    lens = [max(a, b) for a, b in zip(lens, q_lens)]
    lens[7] = q_lens[7] = lens[149] = q_lens[149] = 0
    bt = Batch(sp, rng, lens, q_lens, 2, 64, 16).fill()
    check_attention(sp, rng, bt, 4)


def test_one_long_context_is_split_and_joined(sp):
    rng = np.random.default_rng(10)
    bt = Batch(sp, rng, (20011,), (1,), 2, 128, 64).fill()
    check_attention(sp, rng, bt, 8)
    check_attention(sp, rng, bt, 8, q=(f16(rng, 1, 8, 128) * np.float16(6)), scale=0.5)    # a few keys take everything


def test_rows_without_keys_get_zeros_and_rows_of_nobody_stay(sp):
    """Contexts of length zero, more new tokens than tokens in the cache, rows behind the last sequence."""
    rng = np.random.default_rng(11)
    bt = Batch(sp, rng, (0, 2, 30), (2, 5, 3), 2, 64, 16)
    bt.fill()
    q = dev(f16(rng, 14, 4, 64))
    out = torch.full((14, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, max_q=5, out=out)
    assert not bool(out[:2].any()) and not bool(out[2:5].any()) and bool((out[10:] == 7).all())
    for b, (first, t, skip) in {1: (5, 5, 3), 2: (7, 3, 0)}.items():
        k, v, sc = bt.held(b)
        rows = slice(first, 7) if b == 1 else slice(7, 10)
        want, tol = model.attention(q[rows].cpu().numpy().astype(np.float64), k, v, sc, 0.125)
        assert np.all(np.abs(out[rows].cpu().numpy() - want) <= tol)
    assert sp.device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_garbage_behind_the_context_is_not_seen(sp, D):
    """NaN in the pages behind the last token, and in tokens that only some rows may see."""
    rng = np.random.default_rng(12)
    bt = Batch(sp, rng, (37,), (6,), 2, D, 64)
    bt.cache.pool.view(torch.float16).fill_(float("nan"))
    bt.fill()
    check_attention(sp, rng, bt, 4)
    # token 34 (row 3 is the first to see it) gets NaN values in channels 32..63 of head 0, token 36 an infinite key in head 1
    bt.v[0][34, 0, 40] = np.nan
    bt.k[0][36, 1, 3] = np.inf
    bt.fill()
    q = f16(rng, 6, 4, D)
    out = sp.kv_attention(dev(q), bt.cache, bt.table, bt.kv_lens).cpu().numpy().astype(np.float64)
    k, v, sc = bt.held(0)
    bad = np.zeros((6, 4, D), bool)
    bad[3:, :2, 32:64] = True
    bad[5, 2:] = True
    v[34, 0], sc[34, 0] = np.where(np.isnan(v[34, 0]), 0, v[34, 0]), np.where(np.isnan(sc[34, 0]), 0, sc[34, 0])
    k[36, 1] = np.where(np.isnan(k[36, 1]), 0, k[36, 1])
    want, tol = model.attention(q.astype(np.float64), k, v, sc, D ** -0.5)
    assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()
    assert np.all(np.abs(out - want)[~bad] <= tol[~bad])


def test_extreme_queries_and_values(sp):
    """Queries near the largest fp16 value and near the smallest, values near the largest."""
    rng = np.random.default_rng(13)
    bt = Batch(sp, rng, (200,), (4,), 2, 128, 16)
    bt.v[0] = (rng.uniform(-60000, 60000, bt.v[0].shape)).astype(np.float16)
    bt.fill()
    q = f16(rng, 4, 4, 128)
    q[0] *= np.float16(1e4)
    q[1] *= np.float16(1e-5)
    q[2, :, :64] *= np.float16(1e-4)
    q[3] = 0
    check_attention(sp, rng, bt, 4, q=q, scale=1e-4)


def test_attention_in_a_graph_follows_growing_contexts(sp):
    """One captured step (append, attention), replayed while the lengths on the device grow; on a stream of its own."""
    rng = np.random.default_rng(14)
    B, Hkv, Hq, D, page, steps = 3, 2, 4, 128, 16, 40
    start = [14, 1, 60]
    bt = Batch(sp, rng, [n + steps for n in start], [1] * B, Hkv, D, page)
    lens = i32(start)
    sp.kv_append(bt.cache, dev(np.concatenate([bt.k[b][:n] for b, n in enumerate(start)])),
                 dev(np.concatenate([bt.v[b][:n] for b, n in enumerate(start)])), bt.table, lens, cu_q=i32([0, 14, 15, 75]))
    k = torch.zeros((B, Hkv, D), dtype=torch.float16, device="cuda")
    v, q = torch.zeros_like(k), torch.zeros((B, Hq, D), dtype=torch.float16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        lens.add_(1)
        sp.kv_append(bt.cache, k, v, bt.table, lens)
        return sp.kv_attention(q, bt.cache, bt.table, lens)

    with torch.cuda.stream(stream):
        step()                                  # warm-up: its token is written over below
        lens.sub_(1)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for i in range(steps):
        at = [n + i for n in start]
        qh = f16(rng, B, Hq, D)
        k.copy_(dev(np.stack([bt.k[b][p] for b, p in enumerate(at)])))
        v.copy_(dev(np.stack([bt.v[b][p] for b, p in enumerate(at)])))
        q.copy_(dev(qh))
        graph.replay()
        if i % 13 == 0 or i == steps - 1:
            got = out.cpu().numpy().astype(np.float64)
            for b in range(B):
                kk, vv, sc = bt.held(b)
                want, tol = model.attention(qh[b:b + 1].astype(np.float64), kk[:at[b] + 1], vv[:at[b] + 1], sc[:at[b] + 1], D ** -0.5)
                assert np.all(np.abs(got[b:b + 1] - want) <= tol)
    assert sp.device_status() == 0


def test_same_bits_every_time_and_on_two_streams_at_once(sp):
    rng = np.random.default_rng(15)
    bt = Batch(sp, rng, (3000, 17, 900), (1, 1, 1), 4, 128, 32).fill()
    q = dev(f16(rng, 3, 16, 128))
    first = sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    # a stream given by hand
    other = sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens, stream=streams[0])
    streams[0].synchronize()
    assert torch.equal(other, first)


def test_strided_queries(sp):
    rng = np.random.default_rng(16)
    bt = Batch(sp, rng, (50, 3), (1, 1), 2, 64, 16).fill()
    fused = dev(f16(rng, 2, 8, 64))
    a = sp.kv_attention(fused[:, 2:6], bt.cache, bt.table, bt.kv_lens)
    b = sp.kv_attention(fused[:, 2:6].contiguous(), bt.cache, bt.table, bt.kv_lens)
    assert torch.equal(a, b)


def test_shared_pages(sp):
    """Two sequences with the same first page (a shared prefix) read the same tokens."""
    rng = np.random.default_rng(17)
    bt = Batch(sp, rng, (16 + 5, 16 + 9), (5, 9), 2, 64, 16, spare=2)
    table = bt.table_h.copy()
    table[1, 0] = table[0, 0]
    bt.table = dev(table)
    bt.k[1][:16], bt.v[1][:16] = bt.k[0][:16], bt.v[0][:16]
    sp.kv_append(bt.cache, dev(bt.k[0]), dev(bt.v[0]), bt.table[:1].contiguous(), bt.kv_lens[:1].contiguous())
    sp.kv_append(bt.cache, dev(bt.k[1][16:]), dev(bt.v[1][16:]), bt.table[1:].contiguous(), bt.kv_lens[1:].contiguous())
    check_attention(sp, rng, bt, 4)


def test_offsets_past_the_rows_touch_nothing_behind_them(sp):
    """cu_q says more rows than there are, with enough of them for a warp to take eight: the rows there are count, as the last of the
    sequence, and nothing behind them is written."""
    rng = np.random.default_rng(21)
    heads, D, n, more = 32, 64, 1203, 5
    assert n * 2 * heads >= 8 * 64 * 150 and n % 8
    bt = Batch(sp, rng, [n], [n], heads, D, 64)
    cu = i32([0, n + more])
    sp.kv_append(bt.cache, dev(bt.k[0]), dev(bt.v[0]), bt.table, bt.kv_lens, cu_q=cu)
    whole = [torch.full((n + more, heads, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    sp.kv_read(bt.cache, bt.table, bt.kv_lens, cu_q=cu, k_out=whole[0][:n], v_out=whole[1][:n])
    for got, want in zip(whole, (bt.k[0], bt.v[0])):
        assert np.array_equal(got[:n].cpu().numpy(), model.entry(want.astype(np.float64)).astype(np.float16))
        assert bool((got[n:] == 7).all())
    assert sp.device_status() == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_queries_may_be_turned_and_answered_in_place(sp, interleaved):
    rng = np.random.default_rng(22)
    lens, q_lens, heads, Hq, D = (300, 5, 90), (40, 5, 70), 24, 24, 128
    bt = Batch(sp, rng, lens, q_lens, heads, D, 32).fill()
    n = sum(q_lens)
    cos, sin = (dev(f(np.arange(300)[:, None] * 10000.0 ** (-np.arange(0, 128, 2) / 128)).astype(np.float32)) for f in (np.cos, np.sin))
    k, v, q = (dev(f16(rng, n, h, D)) for h in (heads, heads, Hq))
    args = dict(cu_q=bt.cu, cos=cos, sin=sin, interleaved=interleaved)
    want = sp.kv_append(bt.cache, k, v, bt.table, bt.kv_lens, q=q, **args)
    assert sp.kv_append(bt.cache, k, v, bt.table, bt.kv_lens, q=q, q_out=q, **args) is q or torch.equal(q, want)
    assert torch.equal(q, want)
    for max_q in (70, 1):   # with the kernel for many rows and without
        q = want.clone()
        out = sp.kv_attention(q.clone(), bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, max_q=max_q)
        sp.kv_attention(q, bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, max_q=max_q, out=q)
        assert torch.equal(q, out)
    with pytest.raises(sp.SpmmError, match="overlap"):
        buf = torch.zeros(n * Hq * D + 8, dtype=torch.float16, device="cuda")
        sp.kv_attention(buf[:-8].view(n, Hq, D), bt.cache, bt.table, bt.kv_lens, cu_q=bt.cu, out=buf[8:].view(n, Hq, D))
    assert sp.device_status() == 0


def test_sequences_that_share_rows_beyond_counting_are_refused(sp):
    """cu_q that gives every other sequence all the rows: more units than the list can number."""
    B, n, heads, D = 4000, 64, 64, 64
    cache = sp.KvCacheInt4(1, 16, heads, D)
    table = torch.zeros((B, 60000), dtype=torch.int32, device="cuda")
    lens = torch.full((B,), 60000 * 16, dtype=torch.int32, device="cuda")
    cu = i32([0] + [n if b % 2 == 0 else 0 for b in range(B)])
    q = torch.zeros((n, heads, D), dtype=torch.float16, device="cuda")
    assert heads * (n // 8 + B) * 7500 < 2 ** 31 - 2 ** 25 < 2 ** 31 < B // 2 * heads * (n // 8) * 7500
    out = torch.full_like(q, 7.0)
    sp.kv_attention(q, cache, table, lens, cu_q=cu, max_q=1, out=out)
    assert sp.device_status() & 8
    sp.reset_device_status()
    assert bool((out == 7).all())


def test_cache_is_copied_with_a_handle_of_its_own(sp):
    import copy
    rng = np.random.default_rng(23)
    bt = Batch(sp, rng, (40,), (40,), 2, 64, 16).fill()
    other = copy.deepcopy(bt.cache)
    want = [x.clone() for x in sp.kv_read(bt.cache, bt.table, bt.kv_lens, n_tokens=40)]
    bt.cache.pool.zero_()
    for a, b in zip(sp.kv_read(other, bt.table, bt.kv_lens, n_tokens=40), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,Hkv,group", [(128, 12, 1), (64, 7, 1), (128, 2, 8), (64, 1, 16)])
def test_short_contexts_are_as_exact_as_their_rounding(sp, D, Hkv, group):
    """Over few keys the roundings of the weights do not average out.  What is left in fp32 is below 2^-17 of the output in the root mean
    square (scores of some tens of terms, exponentials to 2^-22), an eightieth of the 2^-11 / sqrt(3) / 1.4 that the rounding to fp16
    makes, which is measured on the exact result: a tenth more is allowed."""
    rng = np.random.default_rng(24)
    lens = [1 + i % 9 for i in range(40)]
    bt = Batch(sp, rng, lens, [1] * 40, Hkv, D, 16).fill()
    q = f16(rng, 40, Hkv * group, D)
    got = sp.kv_attention(dev(q), bt.cache, bt.table, bt.kv_lens).cpu().numpy().astype(np.float64)
    want = np.stack([model.attention(q[b:b + 1].astype(np.float64), *bt.held(b), D ** -0.5)[0][0] for b in range(40)])
    rounding = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)
    assert np.linalg.norm(got - want) <= 1.1 * rounding
    assert sp.device_status() == 0
