"""What the Python calls of the 4-bit operators refuse before anything is launched; no GPU needed."""
import pickle

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def sp(lib_built):
    import spmspm_b200
    return spmspm_b200


def cache_of(sp, pool, num_pages=4, page_size=16, kv_heads=2, head_dim=64):
    """A cache around a pool, as unpickling makes it."""
    c = sp.KvCacheInt4.__new__(sp.KvCacheInt4)
    c.__setstate__(dict(num_pages=num_pages, page_size=page_size, kv_heads=kv_heads, head_dim=head_dim, _pool=pool))
    return c


def calls(sp, cache, table, lens, x):
    """Every call on a cache, with its tensors on their device."""
    return [lambda: sp.kv_append(cache, x, x, table, lens), lambda: sp.kv_read(cache, table, lens, n_tokens=2),
            lambda: sp.kv_attention(x, cache, table, lens), lambda: sp.kv_attention_workspace(cache, 4, 2, 1)]


def test_a_cache_loaded_without_a_device_is_not_used(sp):
    """Saved caches may be loaded on the CPU; with every tensor there the calls would hand host addresses to the kernels."""
    cache = pickle.loads(pickle.dumps(cache_of(sp, torch.zeros(4 * 2 * 1280, dtype=torch.uint8))))
    table, lens, x = torch.zeros((2, 2), dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros((2, 2, 64), dtype=torch.float16)
    for call in calls(sp, cache, table, lens, x):
        with pytest.raises(sp.SpmmError, match="CUDA device"):
            call()


BIG = 1 << 32


@pytest.mark.parametrize("M,K,group", [(BIG + 64, 128, 64), (64, BIG + 128, 64), (64, 128, BIG + 64), (-BIG + 64, 128, 64)])
def test_sizes_are_not_cut_to_32_bits(sp, M, K, group):
    """A size whose low 32 bits fit the data."""
    with pytest.raises(sp.SpmmError, match="out of range"):
        sp.linear_int4(sp.Int4Matrix(M, K, group, torch.zeros(9216, dtype=torch.uint8)), torch.zeros((1, 128), dtype=torch.float16))


def test_workspace_of_sizes_without_one(lib_built):
    """Rows a key head are counted in 64 bits, sizes that no call takes have no workspace."""
    small, large = (lib_built.spb_kv_attention_workspace_bytes(128, 1, 1 << 16, 1, q) for q in (0, 1 << 15))
    assert large == lib_built.spb_kv_attention_workspace_bytes(128, 1, 1 << 16, 1, 1 << 10) != small
