"""What the 4-bit operators refuse, at the C boundary, without a GPU: nothing may be launched for these arguments."""
import ctypes

import pytest

A = 1 << 20          # an aligned address that is never dereferenced: the checks come first


def append(lib, **kw):
    a = dict(stream=None, pool=A, num_pages=4, page_size=16, kv_heads=2, head_dim=64, table=A, stride=2, lens=A, cu=None, batch=2, n=4,
             k=A, kt=128, kh=64, v=A, vt=128, vh=64, q=None, qt=0, qh=0, q_heads=0, q_out=None, cos=None, sin=None, max_pos=0, rot=0, inter=0)
    a.update(kw)
    return lib.spb_kv_append(*a.values())


def attention(lib, **kw):
    a = dict(stream=None, pool=A, num_pages=4, page_size=16, kv_heads=2, head_dim=64, table=A, stride=2, lens=A, cu=None, batch=2, n=4,
             q=A, qt=128, qh=64, q_heads=4, max_q=2, scale=0.1, out=A, ws=A, ws_bytes=1 << 30)
    a.update(kw)
    return lib.spb_kv_attention(*a.values())


COMMON = [dict(head_dim=96), dict(num_pages=0), dict(page_size=8), dict(page_size=24), dict(kv_heads=0), dict(batch=0), dict(batch=70000),
          dict(stride=0), dict(n=-1), dict(n=3), dict(n=1 << 31, cu=A), dict(pool=None), dict(table=None), dict(lens=None), dict(pool=A + 8), dict(table=A + 2),
          dict(lens=A + 1), dict(cu=A + 2)]


@pytest.mark.parametrize("bad", COMMON + [dict(k=None), dict(v=None), dict(k=A + 4), dict(kt=130), dict(vh=-64), dict(cos=A), dict(sin=A),
                                          dict(cos=A, sin=A, max_pos=0, rot=64), dict(cos=A, sin=A, max_pos=9, rot=12),
                                          dict(cos=A, sin=A, max_pos=9, rot=72), dict(cos=A + 2, sin=A, max_pos=9, rot=64),
                                          dict(q=A, q_out=A, q_heads=4), dict(q=A, q_out=None, q_heads=4, cos=A, sin=A, max_pos=9, rot=64),
                                          dict(q=A, q_out=A, q_heads=0, cos=A, sin=A, max_pos=9, rot=64),
                                          dict(q=A, qt=2, q_out=A, q_heads=4, cos=A, sin=A, max_pos=9, rot=64)])
def test_append_refuses(lib_built, bad):
    assert append(lib_built, **bad) != 0 and b"kv_append" in lib_built.spb_last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(q=None), dict(q=A + 4), dict(qt=6), dict(q_heads=3), dict(q_heads=0), dict(max_q=-1), dict(max_q=5),
                                          dict(out=None), dict(out=A + 8), dict(ws=None), dict(ws=A + 4), dict(ws_bytes=64)])
def test_attention_refuses(lib_built, bad):
    assert attention(lib_built, **bad) != 0 and b"kv_attention" in lib_built.spb_last_error()


@pytest.mark.parametrize("bad", COMMON)
def test_read_refuses(lib_built, bad):
    a = dict(stream=None, pool=A, num_pages=4, page_size=16, kv_heads=2, head_dim=64, table=A, stride=2, lens=A, cu=None, batch=2, n=4, k=A, v=A)
    a.update(bad)
    assert lib_built.spb_kv_read(*a.values()) != 0 and b"kv_read" in lib_built.spb_last_error()


def test_no_new_tokens_is_no_launch(lib_built):
    before = lib_built.spb_launch_count()
    assert append(lib_built, n=0) == 0 and attention(lib_built, n=0, max_q=0) == 0
    assert lib_built.spb_launch_count() == before


def test_sizes(lib_built):
    assert lib_built.spb_kv_cache_bytes(3, 32, 2, 128) == 3 * 2 * 2 * 2560
    assert lib_built.spb_kv_cache_bytes(3, 24, 2, 128) == 0 and lib_built.spb_kv_cache_bytes(3, 32, 2, 80) == 0
    assert lib_built.spb_int4_bytes(64, 128, 128) == 8704 and lib_built.spb_int4_bytes(192, 192, 32) == 4 * (8192 + 2048)
    assert lib_built.spb_int4_bytes(64, 192, 128) == 0
    assert lib_built.spb_int4_workspace_bytes(100 * 128, 1, 5120) > 0 and lib_built.spb_int4_workspace_bytes(148 * 128, 1, 5120) == 0


@pytest.mark.parametrize("bad", [dict(M=0), dict(M=100), dict(K=96), dict(group=16), dict(group=256), dict(K=192, group=128), dict(N=0), dict(act=2),
                                 dict(codes=None), dict(x=None), dict(out=None), dict(x=A + 2), dict(bias=A + 8),
                                 dict(residual=A + 4), dict(codes=A + 4), dict(N=40, ws=None), dict(N=40, ws=A, ws_bytes=16),
                                 dict(N=40, ws=A + 4, ws_bytes=1 << 30)])
def test_linear_refuses(lib_built, bad):
    a = dict(stream=None, codes=A, M=64, K=128, group=64, x=A, out=A, N=1, bias=None, residual=None, act=0, ws=A, ws_bytes=1 << 30)
    a.update(bad)
    assert lib_built.spb_linear_int4(*a.values()) != 0 and b"linear_int4" in lib_built.spb_last_error()


def test_pack_encode_decode_refuse(lib_built):
    for M, K, g in ((100, 128, 64), (64, 100, 64), (64, 128, 48), (64, 192, 128)):
        assert lib_built.spb_int4_pack(None, A, A, A, M, K, g, A) != 0
        assert lib_built.spb_int4_encode(None, A, M, K, g, A, A, A) != 0
        assert lib_built.spb_int4_decode(None, A, M, K, g, A) != 0
    assert lib_built.spb_int4_pack(None, None, A, A, 64, 128, 64, A) != 0
    assert lib_built.spb_int4_encode(None, A, 64, 128, 64, None, A, A) != 0
    assert lib_built.spb_int4_decode(None, A, 64, 128, 64, A + 2) != 0


def test_python_wrappers_refuse_before_any_call(lib_built):
    """Tensors of the wrong kind are refused by name, on the CPU, before the library is asked."""
    torch = pytest.importorskip("torch")
    import spmspm_b200 as sp
    for bad in (dict(head_dim=80), dict(page_size=20), dict(num_pages=0), dict(kv_heads=-1)):
        with pytest.raises(sp.SpmmError):
            sp.KvCacheInt4(**{**dict(num_pages=4, page_size=16, kv_heads=2, head_dim=64, device="cpu"), **bad})
    with pytest.raises(sp.SpmmError, match="CUDA"):
        sp.KvCacheInt4(4, 16, 2, 64, device="cpu")
    codes, scales = torch.zeros((64, 128), dtype=torch.uint8), torch.zeros((64, 2), dtype=torch.float16)
    with pytest.raises(sp.SpmmError, match="codes"):
        sp.pack_int4(codes, scales, torch.zeros((64, 2), dtype=torch.uint8))
    with pytest.raises(sp.SpmmError, match="group"):
        sp.pack_int4(codes, scales[:, :1].expand(64, 32), codes)
    with pytest.raises(sp.SpmmError):
        sp.encode_int4(torch.zeros((64, 128), dtype=torch.float16))
    with pytest.raises(sp.SpmmError, match="W.data"):
        sp.linear_int4(sp.Int4Matrix(64, 128, 64, torch.zeros(9216, dtype=torch.uint8)), torch.zeros((1, 128), dtype=torch.float16))


HALF = 2             # bytes of an fp16 element


@pytest.mark.parametrize("bad", [dict(out=A + 16), dict(out=A, qt=512), dict(out=A + HALF * 4 * 256 - 16), dict(q=A + 16, out=A), dict(out=A, qh=128, qt=512)])
def test_attention_refuses_an_output_across_the_queries(lib_built, bad):
    assert attention(lib_built, **{**dict(qt=256, q_heads=4), **bad}) != 0 and b"overlap" in lib_built.spb_last_error()


@pytest.mark.parametrize("bad", [dict(q_out=A + 16), dict(q_out=A, qt=512), dict(q_out=2 * A), dict(q_out=3 * A + 512), dict(q_out=2 * A - 16)])
def test_append_refuses_turned_queries_across_its_inputs(lib_built, bad):
    kw = dict(k=2 * A, v=3 * A, q=A, qt=256, qh=64, q_heads=4, cos=A, sin=A, max_pos=9, rot=64)
    assert append(lib_built, **{**kw, **bad}) != 0 and b"overlap" in lib_built.spb_last_error()


def test_read_refuses_keys_across_values(lib_built):
    for k, v in ((A, A), (A, A + 16), (A + HALF * 4 * 128 - 16, A)):
        assert lib_built.spb_kv_read(None, A, 4, 16, 2, 64, A, 2, A, None, 2, 4, k, v) != 0 and b"overlap" in lib_built.spb_last_error()


@pytest.mark.parametrize("bad", [dict(out=2 * A), dict(out=2 * A + HALF * 3 * 128 - 16), dict(residual=A + 16), dict(bias=A + HALF * 3 * 64 - 16)])
def test_linear_refuses_an_output_across_its_inputs(lib_built, bad):
    a = dict(stream=None, codes=3 * A, M=64, K=128, group=64, x=2 * A, out=A, N=3, bias=None, residual=None, act=0, ws=5 * A, ws_bytes=1 << 30)
    a.update(bad)
    assert lib_built.spb_linear_int4(*a.values()) != 0 and b"overlap" in lib_built.spb_last_error()
