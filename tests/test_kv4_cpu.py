"""CPU: the 4-bit cache's reference against the format's definition, sizes, and what its entry points refuse before any launch."""
import ctypes as C

import numpy as np
import pytest

import ref_kv4 as R

BASE = 1 << 20   # an address that no call gets to use


@pytest.fixture()
def cache(pkg):
    return pkg.Kv4Cache(BASE, 10, 2, 4, 128)


def test_struct_layout_matches_header(pkg):
    assert C.sizeof(pkg.Kv4Cache) == 8 + 8 + 4 * 4 and C.sizeof(pkg.RopeArgs) == 3 * 4 + 6 * 4 + 4 + 8


def test_sizes(lib):
    c = lib.c
    assert c.pb200_kv4_page_bytes(1, 1, 128) == R.chunk_bytes(128) == 9216 and c.pb200_kv4_page_bytes(3, 4, 64) == 12 * R.chunk_bytes(64)
    assert c.pb200_kv4_page_bytes(1, 1, 96) == 0 and c.pb200_kv4_page_bytes(0, 1, 128) == 0 and c.pb200_kv4_page_bytes(1, -1, 128) == 0
    assert c.pb200_kv4_attn_workspace_bytes(32, 8, 128) > 0 and c.pb200_kv4_attn_workspace_bytes(32, 5, 128) == 0 and c.pb200_kv4_attn_workspace_bytes(32, 8, 80) == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_every_number_has_bits_of_its_own(dim):
    kb, ks, vb, vs, ksc, vsc = R.places(dim)
    bits = {(int(b), int(s)) for m in ((kb, ks), (vb, vs)) for b, s in zip(m[0].ravel(), m[1].ravel())}
    assert len(bits) == 2 * R.CELLS * dim and max(b for b, _ in bits) == R.CELLS * dim - 1
    scales = {int(x) for x in np.concatenate((ksc.ravel(), vsc.ravel()))}
    assert len(scales) == 2 * R.CELLS * dim // 32 and min(scales) == R.CELLS * dim and max(scales) == R.chunk_bytes(dim) - 2


@pytest.mark.parametrize("dim", [64, 128])
def test_reference_packs_and_steps(dim):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 2, R.CELLS, dim)) * 10.0 ** rng.integers(-6, 4, (2, 2, R.CELLS, 1))
    (kn, ks), (vn, vs) = R.quantize(x[0]), R.quantize(x[1])
    k, v = R.unpack(R.pack(kn, ks, vn, vs), dim)
    assert np.array_equal(k, R.values(kn, ks)) and np.array_equal(v, R.values(vn, vs))
    step = np.abs(np.repeat(ks, 32, -1))
    # half a step; the scale is rounded by 2^-8 at most, times 8 steps, and the end opposite to the largest number has 7 steps only
    assert np.all(np.abs(k - x[0]) <= step * (1.0 + 2.0 ** -4) + 2.0 ** -24)
    assert np.array_equal(k.astype(np.float16).astype(np.float64), k)


def test_format_of_special_numbers():
    n, s = R.quantize(np.array([np.inf, -np.inf, np.nan] + [1.0] * 29))
    assert s[0] == -2720.0 and list(R.values(n, s)[:3]) == [21760.0, -19040.0, 0.0]
    n, s = R.quantize(np.zeros(32))
    assert s[0] == 0 and np.all(n == 8)
    n, s = R.quantize(np.array([3.0, -3.0] + [0.0] * 30))            # of equal magnitudes the first gives the sign
    assert s[0] == -0.375 and R.values(n, s)[0] == 3.0


def test_cache_is_checked(lib, pkg):
    c = lib.c
    for bad, rc in [(pkg.Kv4Cache(None, 10, 1, 1, 128), -1), (pkg.Kv4Cache(BASE + 8, 10, 1, 1, 128), -1), (pkg.Kv4Cache(BASE, 0, 1, 1, 128), -1), (pkg.Kv4Cache(BASE, 1 << 31, 1, 1, 128), -1),
                    (pkg.Kv4Cache(BASE, 10, 0, 1, 128), -1), (pkg.Kv4Cache(BASE, 10, 1, 0, 128), -1), (pkg.Kv4Cache(BASE, 10, 1, 1, 80), -3), (pkg.Kv4Cache(BASE, 10, 1000, 100, 128), -3)]:
        p = C.byref(bad)
        assert c.pb200_kv4_copy_pages(p, None, None, 0, None) == rc
        assert c.pb200_kv4_compact(p, 1, BASE, 1, BASE, 1, BASE, 1, BASE, 0, None) == rc
        assert c.pb200_kv4_load(p, 0, 0, BASE, 0, BASE, 128, BASE, 128, None) == rc
        assert c.pb200_kv4_attn(p, 0, 0, BASE, 128, 2 * BASE, 128, 1, 1, BASE, BASE, BASE, 1, 1, 1, 0.1, 0, 0, BASE, 1 << 30, None) == rc
        assert c.pb200_kv4_append(p, 0, 0, BASE, 128, BASE, 128, BASE, 128, BASE, 128, 1, 1, BASE, BASE, None, None, 1e-6, None, None) == rc
    assert c.pb200_kv4_copy_pages(None, None, None, 0, None) == -1


def attn_args(cache, **kw):
    a = dict(layer=0, type=0, q=BASE, ldq=512, out=16 * BASE, ldo=512, n_head=4, n_seq=1, q_start=BASE, kv_len=BASE, table=BASE, table_ld=4, n_tokens=3, max_q=3, scale=0.1, window=0,
             first=0, ws=BASE, ws_bytes=1 << 30)
    a.update(kw)
    return [C.byref(cache), *a.values(), None]


@pytest.mark.parametrize("kw", [dict(layer=2), dict(layer=-1), dict(type=8), dict(q=None), dict(out=None), dict(q=BASE + 8), dict(ldq=508), dict(ldq=514), dict(ldo=511), dict(n_head=0),
                                dict(n_head=6), dict(n_seq=-1), dict(q_start=None), dict(kv_len=None), dict(table=None), dict(table_ld=0), dict(n_tokens=-1), dict(max_q=-1),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(first=-1), dict(ws=None), dict(ws=BASE + 4), dict(ws_bytes=8),
                                dict(out=BASE + 1024), dict(out=BASE), dict(type=1, q=BASE + 2)], ids=str)
def test_attention_refuses(lib, cache, kw):
    assert lib.c.pb200_kv4_attn(*attn_args(cache, **kw)) == -1


def test_counts_beyond_31_bits(lib, pkg):
    """What the kernels count in 31 bits: refused where it would not fit, and only there (an address that no call gets to use: what is not refused ends in a launch without a GPU)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on the GPU")
    many = pkg.Kv4Cache(BASE, 1 << 30, 1, 8, 128)
    big = dict(ldq=1024, ldo=1024, n_head=8, out=1 << 50, n_tokens=1 << 20, max_q=1)
    assert lib.c.pb200_kv4_attn(*attn_args(many, n_seq=1 << 16, table_ld=4096, **big)) == -3
    assert lib.c.pb200_kv4_attn(*attn_args(many, n_seq=64, table_ld=4096, **dict(big, max_q=2048))) not in (0, -1, -3)


def test_nothing_to_do_is_no_error(lib, cache):
    for kw in (dict(n_seq=0), dict(n_tokens=0), dict(max_q=0)):
        assert lib.c.pb200_kv4_attn(*attn_args(cache, **kw)) == 0
    p = C.byref(cache)
    assert lib.c.pb200_kv4_copy_pages(p, None, None, 0, None) == 0
    assert lib.c.pb200_kv4_compact(p, 0, BASE, 1, BASE, 1, BASE, 1, BASE, 1, None) == 0
    assert lib.c.pb200_kv4_compact(p, 1, BASE, 1, BASE, 1, BASE, 1, BASE, 0, None) == 0
    assert lib.c.pb200_kv4_load(p, 0, 0, BASE, 0, BASE, 512, BASE, 512, None) == 0
    assert lib.c.pb200_kv4_append(*append_args(cache, None, n_tokens=0)) == 0


def append_args(cache, rope, **kw):
    a = dict(layer=0, type=0, q=BASE, ldq=512, q_out=16 * BASE, ldqo=512, k=32 * BASE, ldk=512, v=48 * BASE, ldv=512, n_tokens=3, n_head=4, cells=BASE, pos=BASE, qw=None, kw=None, eps=1e-6)
    a.update(kw)
    return [C.byref(cache), *a.values(), None if rope is None else C.byref(rope), None]


@pytest.mark.parametrize("kw", [dict(layer=2), dict(type=2), dict(q=None), dict(q_out=None), dict(k=None), dict(v=BASE + 4), dict(ldk=508), dict(ldv=513), dict(n_tokens=-1), dict(n_head=-1),
                                dict(cells=None), dict(qw=BASE + 4), dict(kw=BASE + 8), dict(kw=BASE, eps=-1.0), dict(kw=BASE, eps=float("nan")), dict(q_out=BASE + 16),
                                dict(q_out=BASE, ldqo=516)], ids=str)
def test_append_refuses(lib, cache, kw):
    assert lib.c.pb200_kv4_append(*append_args(cache, None, **kw)) == -1


@pytest.mark.parametrize("kw,rc", [(dict(n_dims=136), -1), (dict(n_dims=-8), -1), (dict(n_dims=12), -3), (dict(mode=1), -1), (dict(freq_base=0.0), -1), (dict(freq_scale=0.0), -1)], ids=str)
def test_append_refuses_rotations(lib, pkg, cache, kw, rc):
    a = dict(n_dims=64, mode=2, n_ctx_orig=4096, freq_base=1e4, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0)
    a.update(kw)
    assert lib.c.pb200_kv4_append(*append_args(cache, pkg.RopeArgs(**a))) == rc
    a.update(n_dims=64, mode=2, freq_base=1e4, freq_scale=1.0)
    assert lib.c.pb200_kv4_append(*append_args(cache, pkg.RopeArgs(**a), pos=None)) == -1


def test_load_refuses(lib, cache):
    p, f = C.byref(cache), lib.c.pb200_kv4_load
    for a in [(2, 0, BASE, 1, BASE, 512, BASE, 512), (0, 7, BASE, 1, BASE, 512, BASE, 512), (0, 0, None, 1, BASE, 512, BASE, 512), (0, 0, BASE, -1, BASE, 512, BASE, 512),
              (0, 0, BASE, 1, None, 512, None, 512), (0, 0, BASE, 1, BASE + 4, 512, None, 0), (0, 0, BASE, 1, BASE, 508, None, 0), (0, 1, BASE, 1, None, 0, BASE, 514)]:
        assert f(p, *a, None) == -1, a


def test_copies_have_no_order(lib, cache):
    def rc(src, dst):
        s, d = np.array(src, np.int32), np.array(dst, np.int32)
        return lib.c.pb200_kv4_copy_pages(C.byref(cache), s.ctypes.data, d.ctypes.data, len(src), None)
    assert rc([0, 1], [2, 2]) == -1 and rc([0, 2], [2, 3]) == -1 and rc([1], [1]) == -1 and rc([0], [10]) == -1 and rc([-1], [3]) == -1 and rc([10], [3]) == -1 and rc([3], [-1]) == -1
    assert lib.c.pb200_kv4_copy_pages(C.byref(cache), None, BASE, 1, None) == -1 and lib.c.pb200_kv4_copy_pages(C.byref(cache), None, None, -1, None) == -1


@pytest.mark.parametrize("a", [(-1, BASE, 1, BASE, 1, BASE, 1, BASE, 1), (70000, BASE, 1, BASE, 1, BASE, 1, BASE, 1), (1, None, 1, BASE, 1, BASE, 1, BASE, 1), (1, BASE, 0, BASE, 1, BASE, 1, BASE, 1),
                               (1, BASE, 1, None, 1, BASE, 1, BASE, 1), (1, BASE, 1, BASE, 0, BASE, 1, BASE, 1), (1, BASE, 1, BASE, 1, None, 1, BASE, 1), (1, BASE, 1, BASE, 1, BASE, 1, BASE, 2),
                               (1, BASE, 1, BASE, 1, BASE, 1, None, 1), (1, BASE, 1, BASE, 1, BASE, 1, BASE, -1)], ids=str)
def test_compact_refuses(lib, cache, a):
    assert lib.c.pb200_kv4_compact(C.byref(cache), *a, None) == -1


def test_rows_may_lie_between_each_other(lib, pkg, cache):
    """Refused where a row that is read and one that is written have a number in common, and with equal strides only there (what is not refused ends in a launch without a GPU)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would run on the GPU")
    at, n = 4 << 20, 3
    for ld in (512, 520, 1024, 1536):
        for off in sorted({x for r in range(-n - 1, n + 2) for x in (r * ld, r * ld - 512, r * ld + 512, r * ld - 508, r * ld + 508, r * ld + ld // 8 * 4)}):
            common = any(abs(off + (j - i) * ld) < 512 for i in range(n) for j in range(n))
            rc = lib.c.pb200_kv4_attn(*attn_args(cache, q=at, ldq=ld, out=at + 4 * off, ldo=ld))
            assert (rc == -1) == common and rc != 0, (ld, off)
            for what in ("k", "v"):
                rc = lib.c.pb200_kv4_append(*append_args(cache, None, q=1 << 30, ldq=ld, **{what: at, "ld" + what: ld}, q_out=at + 4 * off, ldqo=ld))
                assert (rc == -1) == common and rc != 0, (what, ld, off)
            rc = lib.c.pb200_kv4_append(*append_args(cache, None, q=at, ldq=ld, q_out=at + 4 * off, ldqo=ld))
            assert (rc == -1) == (common and off != 0) and rc != 0, (ld, off)
    # other strides: ranges apart; a single row has none
    assert lib.c.pb200_kv4_attn(*attn_args(cache, q=at, ldq=1024, out=at + 4 * 512, ldo=2048)) == -1
    assert lib.c.pb200_kv4_attn(*attn_args(cache, q=at, ldq=1024, out=at + 4 * 512, ldo=2048, n_tokens=1)) not in (0, -1, -3)
