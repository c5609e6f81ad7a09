"""The operators around the 4-bit cache: what their entry points refuse, and calls with nothing to do.  No GPU: addresses are never used."""
import ctypes as C

import numpy as np
import pytest

import ref_serve as V

BASE = 1 << 20
BAD = [dict(layer=2), dict(layer=-1), dict(type=8), dict(q=BASE + 8), dict(ldq=508), dict(ldq=514), dict(n_head=0), dict(n_head=6), dict(n_seq=-1), dict(q_start=None), dict(kv_len=None),
       dict(table=None), dict(table_ld=0), dict(n_tokens=-1), dict(max_q=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(type=1, q=BASE + 2)]


@pytest.fixture(scope="module")
def cache(pkg):
    return pkg.Kv4Cache(BASE, 10, 2, 4, 128)


def args(cache, base, **kw):
    a = dict(base)
    a.update(kw)
    return [C.byref(cache), *a.values(), None]


LSE = dict(layer=0, type=0, q=BASE, ldq=512, out=16 * BASE, ldo=512, n_head=4, n_seq=1, q_start=BASE, kv_len=BASE, table=BASE, table_ld=4, n_tokens=3, max_q=3, scale=0.1, window=0, first=0,
           lse=BASE, ld_lse=4, ws=BASE, ws_bytes=1 << 30)
SHARED = dict(layer=0, type=0, q=BASE, ldq=512, out=16 * BASE, ldo=512, n_head=4, n_seq=1, q_start=BASE, kv_len=BASE, table=BASE, table_ld=4, n_group=1, group_start=BASE, prefix_len=BASE,
              prefix_table=BASE, prefix_ld=3, n_tokens=3, max_q=3, scale=0.1, lse=BASE, ld_lse=4, ws=BASE, ws_bytes=1 << 30)
WEIGH = dict(layer=0, type=0, q=BASE, ldq=512, n_head=4, n_seq=3, q_start=BASE, kv_len=BASE, table=BASE, table_ld=4, n_tokens=3, max_q=3, scale=0.1, window=0, first=0, lse=BASE, ld_lse=4,
             decay=0.5, old=BASE, ld_old=256, sums=16 * BASE, ld_sums=256)
SELECT = dict(n_seq=3, sums=BASE, ld_sums=500, kv_len=BASE, max_len=400, budget=BASE, first=4, last=4, index=BASE, ld_index=100, count=BASE, kept=16 * BASE, ld_kept=100)
VERIFY = dict(type=0, target=BASE, ld_target=1000, draft=BASE, ld_draft=1000, n_vocab=1000, n_seq=3, start=BASE, n_drafts=5, tokens=BASE, inv_temp=BASE, u=BASE, v=BASE, accepted=BASE, out=BASE,
              ld_out=4, kv_len=BASE, kv_len_out=BASE, ws=BASE, ws_bytes=1 << 20)


@pytest.mark.parametrize("kw", BAD + [dict(out=None), dict(ldo=511), dict(window=-1), dict(first=-1), dict(ws=None), dict(ws=BASE + 4), dict(ws_bytes=8), dict(out=BASE + 1024), dict(out=BASE),
                                      dict(lse=None), dict(lse=BASE + 2), dict(ld_lse=3)], ids=str)
def test_attention_with_logarithms_refuses(lib, cache, kw):
    assert lib.c.pb200_kv4_attn_lse(*args(cache, LSE, **kw)) == -1


@pytest.mark.parametrize("kw", BAD + [dict(out=None), dict(ldo=511), dict(ws=None), dict(ws=BASE + 4), dict(out=BASE + 1024), dict(lse=BASE + 2), dict(ld_lse=3), dict(n_group=-1),
                                      dict(group_start=None), dict(prefix_len=None), dict(prefix_table=None), dict(prefix_ld=0)], ids=str)
def test_attention_behind_prefixes_refuses(lib, cache, kw):
    assert lib.c.pb200_kv4_attn_shared(*args(cache, SHARED, **kw)) == -1


def test_workspace_of_attention_behind_prefixes(lib, cache):
    c = lib.c
    least = c.pb200_kv4_attn_shared_workspace_bytes(4, 4, 128, 3)
    assert least >= c.pb200_kv4_attn_workspace_bytes(4, 4, 128) + 3 * 4 * (128 * 4 + 8)
    assert c.pb200_kv4_attn_shared(*args(cache, SHARED, ws_bytes=least - 1)) == -1
    assert c.pb200_kv4_attn_shared(*args(cache, SHARED, ws_bytes=c.pb200_kv4_attn_workspace_bytes(4, 4, 128))) == -1
    assert c.pb200_kv4_attn_shared_workspace_bytes(4, 3, 128, 3) == 0 and c.pb200_kv4_attn_shared_workspace_bytes(4, 4, 96, 3) == 0 and c.pb200_kv4_attn_shared_workspace_bytes(4, 4, 128, -1) == 0


@pytest.mark.parametrize("kw", BAD + [dict(q=None), dict(lse=None), dict(lse=BASE + 2), dict(ld_lse=3), dict(window=-1), dict(first=-1), dict(decay=float("nan")), dict(decay=float("inf")), dict(sums=None),
                                      dict(sums=BASE + 1), dict(ld_sums=0), dict(old=BASE + 2), dict(ld_old=255), dict(sums=BASE + 4), dict(sums=BASE + 1024), dict(sums=BASE, ld_old=260)], ids=str)
def test_weights_refuse(lib, cache, kw):
    assert lib.c.pb200_kv4_weigh(*args(cache, WEIGH, **kw)) == -1


@pytest.mark.parametrize("kw", [dict(n_seq=-1), dict(sums=None), dict(sums=BASE + 2), dict(ld_sums=0), dict(kv_len=None), dict(max_len=-1), dict(budget=None), dict(first=-1), dict(last=-1), dict(index=None),
                                dict(ld_index=0), dict(count=None), dict(kept=BASE), dict(kept=BASE + 2), dict(kept=BASE + 4 * 1399), dict(ld_kept=99), dict(kept=BASE - 4 * 299)], ids=str)
def test_selection_refuses(lib, kw):
    assert lib.c.pb200_kv4_select(*{**SELECT, **kw}.values(), None) == -1


@pytest.mark.parametrize("kw", [dict(type=8), dict(target=None), dict(target=BASE + 2), dict(ld_target=999), dict(draft=BASE + 2), dict(ld_draft=999), dict(n_vocab=0), dict(n_vocab=-5), dict(n_seq=-1),
                                dict(start=None), dict(n_drafts=-1), dict(tokens=None), dict(u=None), dict(v=None), dict(accepted=None), dict(out=None), dict(ld_out=0), dict(kv_len=None),
                                dict(kv_len_out=None), dict(ws=None), dict(ws=BASE + 8), dict(ws_bytes=100), dict(type=1, target=BASE + 1)], ids=str)
def test_verification_refuses(lib, kw):
    assert lib.c.pb200_verify_drafts(*{**VERIFY, **kw}.values(), None) == -1


def test_nothing_to_do_is_no_error(lib, cache):
    c = lib.c
    for kw in (dict(n_seq=0), dict(n_tokens=0), dict(max_q=0)):
        assert c.pb200_kv4_attn_lse(*args(cache, LSE, **kw)) == 0 and c.pb200_kv4_attn_shared(*args(cache, SHARED, **kw)) == 0
    assert c.pb200_kv4_weigh(*args(cache, WEIGH, n_seq=0)) == 0
    assert c.pb200_kv4_select(*{**SELECT, "n_seq": 0}.values(), None) == 0
    assert c.pb200_verify_drafts(*{**VERIFY, "n_seq": 0}.values(), None) == 0


def test_sizes_beyond_the_kernels_counts(lib, cache, pkg):
    c = lib.c
    assert c.pb200_verify_drafts(*{**VERIFY, "n_vocab": (1 << 30) + 1, "ld_target": 1 << 31, "ld_draft": 1 << 31}.values(), None) == -3
    assert c.pb200_kv4_select(*{**SELECT, "n_seq": 1 << 30, "kept": None}.values(), None) == -3
    assert c.pb200_kv4_weigh(*args(cache, WEIGH, n_seq=1 << 20, ld_sums=1 << 20, old=None)) == -3
    many = pkg.Kv4Cache(BASE, 1 << 30, 1, 8, 128)
    big = dict(ldq=1024, ldo=1024, n_head=8, out=1 << 50, n_tokens=1 << 20, max_q=1, n_seq=1, ld_lse=8, ws_bytes=1 << 50)
    assert c.pb200_kv4_attn_shared(*args(many, SHARED, **dict(big, n_seq=1 << 16, n_group=1 << 16, prefix_ld=1 << 12))) == -3
    assert c.pb200_kv4_attn_shared(*args(cache, SHARED, n_group=(1 << 24) + 1)) == -3


def test_reference_of_verification_keeps_the_targets_distribution():
    """What comes out of a draft that is verified has the target's distribution, whatever the draft's: counted over an even grid of both random numbers."""
    rng = np.random.default_rng(5)
    target, draft = rng.standard_normal((2, 6)), rng.standard_normal((1, 6))
    p, q = V.softmax(target[0], 1.0), V.softmax(draft[0], 1.0)
    grid = (np.arange(200) + 0.5) / 200
    seen = np.zeros(6)
    for x in range(6):
        for u in grid:
            if u * q[x] < p[x]:
                seen[x] += q[x] / 200
            else:
                for v in grid[::10]:
                    seen[V.verify(target, draft, [x], 1.0, [u], v)[1]] += q[x] / 200 / 20
    # a step of u is 1 / 200 of q: what is accepted of a token, and what is rejected in all, is off by as much at most; a step of v is 1 / 20 of what is rejected, and a token's part of it is off by one
    rejected = np.maximum(q - p, 0.0).sum()
    assert np.abs(seen - p).max() <= 2 / 200 + (rejected + 1 / 200) / 20
