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
