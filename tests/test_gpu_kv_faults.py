"""The paged 4-bit cache on the GPU where calls once went wrong: tokens that are skipped, small values, wide page tables, codes next to a
border."""
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


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def randn(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


@pytest.mark.parametrize("kv_heads,q_heads,D", [(2, 4, 64), (24, 40, 128)])
@pytest.mark.parametrize("length,angles", [(9, 6), (3, 64), (9, 1)])
def test_a_token_without_a_place_or_angles_is_skipped_whole(sp, kv_heads, q_heads, D, length, angles):
    """Seven new tokens of a context of `length` and angles for the first `angles` positions: those before position 0 and those past
    the angles leave pool and q_out as they were, the others are there."""
    rng = np.random.default_rng(length + angles + D)
    n, page = 7, 16
    k, v, q = randn(rng, n, kv_heads, D), randn(rng, n, kv_heads, D), randn(rng, n, q_heads, D)
    pos = np.arange(length - n, length)
    ang = np.arange(angles)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    there = (pos >= 0) & (pos < angles)
    cache = sp.KvCacheInt4(2, page, kv_heads, D)
    table = i32(1).view(1, 1)

    # what the pool and q_out should be: the tokens that are there, one call each, over the same old contents
    cache.pool.fill_(0xA5)
    for i in np.flatnonzero(there):
        sp.kv_append(cache, dev(k[i:i + 1]), dev(v[i:i + 1]), table, i32(pos[i] + 1), q=dev(q[i:i + 1]), cos=dev(cos), sin=dev(sin))
    want = cache.pool.clone()
    assert sp.device_status() == 0

    cache.pool.fill_(0xA5)
    q_out = torch.full((n, q_heads, D), 7.0, dtype=torch.float16, device="cuda")
    sp.kv_append(cache, dev(k), dev(v), table, i32(length), q=dev(q), cos=dev(cos), sin=dev(sin), q_out=q_out)
    assert torch.equal(cache.pool, want)
    got = q_out.cpu().numpy()
    turned = model.rotate(q[there].astype(np.float64), pos[there], cos, sin, False).astype(np.float16)
    assert np.array_equal(got[there], turned) and np.all(got[~there] == 7)
    assert sp.device_status() == (8 if (pos >= angles).any() else 0)
    sp.reset_device_status()


@pytest.mark.parametrize("D,heads", [(128, 24), (64, 40)])
def test_prompt_attention_before_products_that_take_tensor_memory(sp, D, heads):
    """Attention of a prompt, and right behind it kernels that take tensor memory before they wait for it: the same bits as one by one."""
    rng = np.random.default_rng(D)
    n, hidden = 600, heads * D
    cache = sp.KvCacheInt4(2 * 16, 64, heads, D)
    table = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    q, k, v = (dev(randn(rng, 2 * n, heads, D)) for _ in range(3))
    sp.kv_append(cache, k, v, table, i32(n, n))
    dense = dev(randn(rng, 640, hidden) * np.float16(0.02))
    Q, W = sp.encode_int4(dense, 64), sp.encode_device(dense)
    few = dev(randn(rng, 8, hidden))

    def step(wait):
        out = []
        for follow in (lambda x: sp.linear_int4(Q, x[:300].contiguous()), lambda x: sp.spmm(W, few, split_k=1), lambda x: sp.linear_int4(Q, few)):
            x = sp.kv_attention(q, cache, table, i32(n, n)).flatten(1)
            if wait:
                torch.cuda.synchronize()
            out += [x, follow(x)]
            if wait:
                torch.cuda.synchronize()
        return out

    want = step(True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(False), want))
    assert sp.device_status() == 0


def cached(sp, k, v, page=64, capacity=0):
    """One sequence with keys and values [L, heads, D] in a cache; the page table holds `capacity` tokens at least."""
    L, heads, D = k.shape
    pages = -(-L // page)
    cache = sp.KvCacheInt4(pages, page, heads, D)
    table = np.full((1, max(pages, -(-capacity // page))), -1, np.int32)
    table[0, :pages] = np.arange(pages)
    sp.kv_append(cache, dev(k), dev(v), dev(table), i32(L))
    return cache, dev(table), i32(L)


def held(k, v):
    return [f(x.astype(np.float64)) for f, x in ((model.entry, k), (model.entry, v), (model.scaled_codes, v))]


def one_key_apart(D, heads, spread, length, gap):
    """q, k, v and a scale: one key's weight is 2^gap times that of each other, about."""
    rng = np.random.default_rng(int(gap + D + length))
    k = (rng.standard_normal((length, heads, D)) * 0.05).astype(np.float16)
    v = (rng.standard_normal((length, heads, D)) * spread).astype(np.float16)
    q = (rng.standard_normal((1, heads, D)) * 0.1).astype(np.float16)
    q[0, :, 0], k[:, :, 0] = 1, 1
    k[length // 3, :, 0] = 16
    return q, k, v, gap * np.log(2) / 15


def relative_attention(q, k, v, scale):
    """model.attention, with what lies below the fp16 range counted relative to the values: products of weights and scales are taken in
    units of 1 to 2 times the group's largest scale s (2^-15 if that is more), 2^-32 of the largest weight times 15 of those a key; the
    output loses 2^-25 below the smallest normal fp16 value."""
    kk, vv, sc = held(k, v)
    q = q.astype(np.float64)
    want, tol = model.attention(q, kk, vv, sc, scale)
    group = q.shape[1] // kk.shape[1]
    for h in range(q.shape[1]):
        z = kk[:, h // group] @ q[:, h].T * scale
        total = np.exp(z - z.max(0)).sum(0)[:, None]
        s = np.maximum(sc[:, h // group].max() / 15, 2.0 ** -15)
        tol[:, h] += len(kk) / total * 15 * 2.0 ** -32 * (2 * s - 1) + 2.0 ** -25 - 2.0 ** -24
    return want, tol


@pytest.mark.parametrize("D,heads", [(64, 2), (128, 1)])
@pytest.mark.parametrize("spread,length,gap", [(1e-3, 60000, 18), (1e-3, 200000, 19), (1e-4, 60000, 16), (1.0, 60000, 17), (30.0, 60000, 14),
                                               (1e-3, 300, 9), (3000.0, 9000, 10)])
def test_small_values_keep_their_bits(sp, D, heads, spread, length, gap):
    """One key takes the most weight, all others 2^-gap of it, together about as much: what they add to their groups' minima has to
    survive whatever the values' magnitude."""
    q, k, v, scale = one_key_apart(D, heads, spread, length, gap)
    cache, table, lens = cached(sp, k, v)
    got = sp.kv_attention(dev(q), cache, table, lens, scale=scale).cpu().numpy().astype(np.float64)
    want, tol = relative_attention(q, k, v, scale)
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    assert sp.device_status() == 0


def test_groups_of_very_different_magnitude(sp):
    """Groups of one head 2^12 apart, and scales of one group that grow along the context."""
    q, k, v, scale = one_key_apart(128, 1, 1.0, 30000, 15)
    v = (v.astype(np.float64) * np.repeat([1e-3, 4.0, 30.0, 3e-4], 32)).astype(np.float16)
    cache, table, lens = cached(sp, k, v)
    got = sp.kv_attention(dev(q), cache, table, lens, scale=scale).cpu().numpy().astype(np.float64)
    for g in range(4):
        cut = slice(32 * g, 32 * g + 32)
        one = np.zeros_like(v)
        one[:, :, cut] = v[:, :, cut]
        want, tol = relative_attention(q, k, one, scale)
        assert np.all(np.abs(got - want)[:, :, cut] <= tol[:, :, cut]), g
    v = (v.astype(np.float64) * (2.0 ** (12 * np.arange(30000) / 30000 - 8))[:, None, None]).astype(np.float16)
    cache, table, lens = cached(sp, k, v)
    got = sp.kv_attention(dev(q), cache, table, lens, scale=scale).cpu().numpy().astype(np.float64)
    want, tol = relative_attention(q, k, v, scale)
    assert np.all(np.abs(got - want) <= tol)
    assert sp.device_status() == 0


def ragged(sp, rng, lens, heads, D, page, capacity):
    """Sequences of given lengths in a cache whose table holds `capacity` tokens of each."""
    width = -(-max(capacity, *lens) // page)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for b, n in enumerate(lens):
        pages = -(-n // page)
        table[b, :pages] = np.arange(at, at + pages)
        at += pages
    cache = sp.KvCacheInt4(at, page, heads, D)
    k, v = ([randn(rng, n, heads, D) for n in lens] for _ in range(2))
    cu = i32(0, *np.cumsum(lens))
    sp.kv_append(cache, dev(np.concatenate(k)), dev(np.concatenate(v)), dev(table), i32(*lens), cu_q=cu)
    return cache, dev(table), i32(*lens), k, v


def off_by(got, want):
    """Errors and the rounding of the exact result to fp16, in the root mean square; what is left in fp32 is a hundredth of it."""
    return np.linalg.norm(got - want), np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)


@pytest.mark.parametrize("D,heads,group", [(128, 12, 1), (64, 7, 1), (128, 2, 8), (64, 1, 16)])
def test_short_contexts_in_wide_tables(sp, D, heads, group):
    """Contexts of a few tokens are as exact in a table made for long ones, and beside a long one; and give the same bits."""
    rng = np.random.default_rng(D + heads)
    lens = [1 + i % 9 for i in range(40)]
    cache, table, n, k, v = ragged(sp, rng, lens, heads, D, 16, 0)
    q = randn(rng, 41, heads * group, D)
    narrow = sp.kv_attention(dev(q[:40]), cache, table, n)
    want = np.concatenate([model.attention(q[b:b + 1].astype(np.float64), *held(k[b], v[b]), D ** -0.5)[0] for b in range(40)])
    for capacity in (129, 600, 40000):
        wide = torch.full((40, -(-capacity // 16)), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        got = sp.kv_attention(dev(q[:40]), cache, wide, n)
        err, rounding = off_by(got.cpu().numpy().astype(np.float64), want)
        assert err <= 1.1 * rounding, capacity
        assert torch.equal(got, narrow), capacity
    cache, table, n, k, v = ragged(sp, rng, lens + [5000], heads, D, 16, 0)
    want = np.concatenate([model.attention(q[b:b + 1].astype(np.float64), *held(k[b], v[b]), D ** -0.5)[0] for b in range(40)])
    err, rounding = off_by(sp.kv_attention(dev(q), cache, table, n)[:40].cpu().numpy().astype(np.float64), want)
    assert err <= 1.1 * rounding
    assert sp.device_status() == 0


def test_the_first_rows_of_a_prompt_are_as_exact_as_their_rounding(sp):
    """A prompt of more than one unit of the context, too few heads for the kernel for many rows: rows that see a few keys."""
    rng = np.random.default_rng(31)
    D, heads, n = 128, 6, 200
    cache, table, lens, k, v = ragged(sp, rng, [n], heads, D, 32, 0)
    q = randn(rng, n, heads, D)
    got = sp.kv_attention(dev(q), cache, table, lens).cpu().numpy().astype(np.float64)
    want = model.attention(q.astype(np.float64), *held(k[0], v[0]), D ** -0.5)[0]
    err, rounding = off_by(got[:16], want[:16])
    assert err <= 1.1 * rounding


@pytest.mark.parametrize("D", [64, 128])
def test_codes_next_to_a_border(sp, D):
    """Values whose difference from the group's minimum does not fit in 32 bits, at and next to the middle between two codes, and groups of
    ordinary and tiny values: the codes are those of the exact quotient."""
    rng = np.random.default_rng(D)
    heads, n = 8, 4000
    x = (rng.standard_normal((n, heads, D)) * np.repeat([1, 30, 1000, 8000], 2)[:, None]).clip(-60000, 60000).astype(np.float16)
    x[:, :, 5:12] = (rng.standard_normal((n, heads, 7)) * 1e-5).astype(np.float16)
    for i in range(1500):   # a range of 15 codes of s, a power of two, that ends k + 1/2 codes below zero
        s, k = 2.0 ** rng.integers(-8, 10), rng.integers(0, 15)
        x[i, :, :32] = 0
        x[i, :, 0], x[i, :, 1] = -(k + 0.5) * s, (14.5 - k) * s
        x[i, :, 2:32] = (rng.choice([-1, 0, 1], (heads, 30)) * 2.0 ** rng.integers(-24, -8, (heads, 30))).astype(np.float16)
    cache = sp.KvCacheInt4(-(-n // 64), 64, heads, D)
    table = torch.arange(-(-n // 64), dtype=torch.int32, device="cuda").view(1, -1)
    sp.kv_append(cache, dev(x), dev(x), table, i32(n))
    want = model.entry(x.astype(np.float64)).astype(np.float16)
    with np.errstate(invalid="ignore"):   # what the quotient of the difference rounded to 32 bits would give: the inputs tell
        g = x.reshape(n, heads, -1, 32).astype(np.float32)
        s = model.quantise(x.astype(np.float64))[1].astype(np.float32)
        rounded = np.clip(np.rint((g - g.min(-1, keepdims=True)) / s), 0, 15)
        assert (rounded != model.quantise(x.astype(np.float64))[0]).sum() > 10000
    for got in sp.kv_read(cache, table, i32(n), n_tokens=n):
        assert np.array_equal(got.cpu().numpy(), want)
    assert sp.device_status() == 0


@pytest.mark.parametrize("heads,group,D", [(2, 4, 64), (3, 1, 128), (1, 20, 64)])
@pytest.mark.parametrize("batch,most", [(300, 900), (1100, 260), (40, 6000)])
def test_many_ragged_sequences_with_and_without_a_bound(sp, heads, group, D, batch, most):
    """Row tiles cut between thread blocks in every way: long and short contexts, sequences without new tokens, few and many parts."""
    rng = np.random.default_rng(batch + heads + D)
    lens = [int(n) for n in np.exp(rng.uniform(0, np.log(most), batch))]
    new = [min(n, int(t)) for n, t in zip(lens, rng.integers(0, 4, batch))]
    lens[5] = new[5] = 0
    lens[batch // 2] = most
    cache, table, n, k, v = ragged(sp, rng, lens, heads, D, 16, 2 * most)
    q = randn(rng, sum(new), heads * group, D)
    cu = i32(0, *np.cumsum(new))
    first = np.cumsum([0] + new)
    for max_q in (3, None):
        got = sp.kv_attention(dev(q), cache, table, n, cu_q=cu, max_q=max_q).cpu().numpy().astype(np.float64)
        for b in [*rng.integers(0, batch, 25), batch // 2, batch - 1, 0]:
            rows = slice(first[b], first[b + 1])
            if new[b]:
                want, tol = model.attention(q[rows].astype(np.float64), *held(k[b], v[b]), D ** -0.5)
                assert np.all(np.abs(got[rows] - want) <= tol), (b, max_q)
    assert sp.device_status() == 0


def test_a_table_far_wider_than_the_contexts(sp):
    """Room for 2^29 tokens and a few thousand of them: what counts is the contexts."""
    rng = np.random.default_rng(41)
    D, heads, group, page = 64, 2, 8, 65536
    k, v = randn(rng, 900, heads, D), randn(rng, 900, heads, D)
    cache = sp.KvCacheInt4(1, page, heads, D)
    narrow = i32(0).view(1, 1)
    wide = torch.full((1, 8192), -1, dtype=torch.int32, device="cuda")
    wide[0, 0] = 0
    sp.kv_append(cache, dev(k), dev(v), wide, i32(900))
    q = randn(rng, 700, heads * group, D)
    want, tol = model.attention(q.astype(np.float64), *held(k, v), D ** -0.5)
    for table in (narrow, wide):
        got = sp.kv_attention(dev(q), cache, table, i32(900), cu_q=i32(0, 700), max_q=1).cpu().numpy().astype(np.float64)
        assert np.all(np.abs(got - want) <= tol)
    # also with the kernel for many rows beside the other
    cache = sp.KvCacheInt4(1, page, 24, D)
    k, v, q = (randn(rng, 900, 24, D) for _ in range(3))
    sp.kv_append(cache, dev(k), dev(v), wide, i32(900))
    table = wide.repeat(2, 1)
    args = dict(cu_q=i32(0, 850, 900), max_q=850)
    assert torch.equal(sp.kv_attention(dev(q), cache, table, i32(900, 50), **args), sp.kv_attention(dev(q), cache, narrow.repeat(2, 1), i32(900, 50), **args))
    assert sp.device_status() == 0


@pytest.mark.parametrize("rows", [1, 3])
def test_nan_in_the_middle_of_a_context_stays_in_its_group(sp, rows):
    """A value that is not finite in one group of one token that every row sees, and scales that grow behind it."""
    rng = np.random.default_rng(51)
    D, heads, L = 128, 2, 3000
    k, v = randn(rng, L, heads, D), randn(rng, L, heads, D)
    v[2000:] *= np.float16(40)
    bad = v.copy()
    bad[700, 1, 70] = np.inf
    q = randn(rng, rows, heads * 4, D)
    cache, table, lens = cached(sp, k, bad)
    got = sp.kv_attention(dev(q), cache, table, lens).cpu().numpy().astype(np.float64)
    want, tol = model.attention(q.astype(np.float64), *held(k, v), D ** -0.5)
    lost = np.zeros(got.shape, bool)
    lost[:, 4:, 64:96] = True
    assert np.isnan(got[lost]).all() and np.all(np.abs(got - want)[~lost] <= tol[~lost])
    assert sp.device_status() == 0
