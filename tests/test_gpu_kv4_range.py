"""The 4-bit cache's operators at the ends of their ranges: counts and lengths that say too much, weights and values many binary orders apart, long prompts, buffers that interleave."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import ref_kv4 as R
from gpu_util import ptr
from test_gpu_kv4 import MIXED, TORCH, Attn, random_pages


pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("q,kv", [([1, 3, 1], [300, 64, 1000]), ([200, 40, 1], [400, 90, 70])], ids=["tokens", "prompts"])
# The root mean square of a rounding, relative to numbers whose logarithms are spread evenly over a binary order: half a step h is h / m of a number m of [1, 2), even over -h .. h, and
# the mean of 1 / m^2 is 3 / (8 ln 2): h * sqrt(0.541 / 3) = 0.4246 h.  16 bits round a weight to f16, BF16 with few rows its product with a scale too, and the output; errors of weights add up
# over cells as the (random) values do, so relative to the output's norm they are what they are relative to a weight.
RMS = {"f16": 0.4246 * 2.0 ** -11 * 2 ** 0.5, "bf16": 0.4246 * (2 * 2.0 ** -22 + 2.0 ** -16) ** 0.5}
ON_THE_WHOLE = {t: 1.1 * r for t, r in RMS.items()}      # a tenth for samples of some thousand numbers


def result(a):
    """(output, what it should be) of the rows of sequences"""
    torch.cuda.synchronize()
    assert a.lib.c.pb200_aborted() == 0
    want = a.want()[0]
    got = a.out[:, :a.heads * a.dim].double().cpu().numpy().reshape(want.shape)
    mine = ~np.isnan(want[:, 0, 0])
    return got[mine], want[mine]


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


# ---------------------------------------------------------------------------------------------------------------- counts and lengths
@pytest.mark.parametrize("layers,kv_heads,dim", [(1, 1, 64), (2, 3, 128)])
def test_compaction_stops_at_its_most(pkg, lib, cuda, layers, kv_heads, dim):
    """Counts above max_count are max_count: the next row's indices, and what lies behind the last row, move nothing (what a count let through would still be cells of the cache)."""
    rng = np.random.default_rng(40)
    n, most, per = 4, 100, 3
    pages_np = random_pages(rng, 2 * n * per, layers * kv_heads, dim)
    order = rng.permutation(2 * n * per).astype(np.int32)
    table, to = order[:n * per].reshape(n, per), order[n * per:].reshape(n, per)
    index = rng.integers(0, per * 64, n * most + 64).astype(np.int32)          # 64 behind the last row
    count = np.array([120, 100, 2 ** 31 - 1, -7], np.int32)
    pages = torch.from_numpy(pages_np).cuda()
    cache = pkg.Kv4Cache(pages.data_ptr(), len(pages_np), layers, kv_heads, dim)
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, to, index, count)]
    lib.check(lib.c.pb200_kv4_compact(C.byref(cache), n, ptr(dev[0]), per, ptr(dev[1]), per, ptr(dev[2]), most, ptr(dev[3]), most, None))
    torch.cuda.synchronize()
    old, want = R.unpack(pages_np, dim), R.unpack(pages_np, dim)
    for s in range(n):
        for i in range(max(0, min(int(count[s]), most))):
            c = index[s * most + i]
            for w, o in zip(want, old):
                w[to[s, i // 64], :, i % 64] = o[table[s, c // 64], :, c % 64]
    assert all(np.array_equal(g, w) for g, w in zip(R.unpack(pages.cpu().numpy(), dim), want))


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("q", [[1, 2], [200, 70]], ids=["tokens", "prompts"])
@pytest.mark.parametrize("pages", [1, 3, 4])
@pytest.mark.parametrize("window,back", [(0, 0), (0, 130), (2 ** 31 - 400, 0)])
def test_lengths_next_to_the_largest_behind_a_short_table(pkg, lib, cuda, type_, q, pages, window, back):
    """Positions up to 2^31 - 2: cells behind the table, and pages that are none, are seen by nobody, whatever the position."""
    a = Attn(pkg, lib, 41, type_, 8, 2, 128, q, [64 * pages] * 2, window=window, extra_cols=0)
    if pages > 1:
        a.table_np[1, 1] = -1
    a.kv_np = np.array([2 ** 31 - 1 - back, 2 ** 31 - 1], np.int32)
    a.upload()
    a.call()
    a.check()
    got, want = result(a)
    if want.any():
        assert off(got, want) <= (1e-5 if type_ == "f32" else ON_THE_WHOLE[type_])


# ---------------------------------------------------------------------------------------------------------------- magnitudes
@pytest.mark.parametrize("gap", [12, 16, 20, 24, 28])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@BOTH
def test_a_cell_ahead_of_all_that_has_no_value(pkg, lib, cuda, type_, gap, q, kv):
    """The first cell's score is `gap` binary orders above the others' and its value is zero: what comes out is the others'.  A weight is off by its own rounding or by 2^-39 of the largest
    (prompts of 16 bits, whose reference may fall behind the largest score by 2^6: 2^-34) at most, evenly spread (root mean square: a sqrt(3)-th); scores of gap * ln 2 by two roundings of 32
    bits."""
    a = Attn(pkg, lib, 42, type_, 8, 2, 128, q, kv, scale=1.0)
    rng = np.random.default_rng(43)
    k, v = rng.standard_normal((2, len(a.pages_np), 2, 64, 128))
    k[..., 0] = 0.0
    for s in range(len(kv)):
        k[a.table_np[s, 0], :, 0], v[a.table_np[s, 0], :, 0] = 0.0, 0.0
        k[a.table_np[s, 0], :, 0, 0] = gap * np.log(2.0)
    a.pages_np = R.pack(*R.quantize(k), *R.quantize(v))
    a.q *= 0.05
    a.q.view(a.tokens, 8, 128)[..., 0] = 1.0
    a.q_np = a.q.double().cpu().numpy()
    a.upload()
    a.call()
    got, want = result(a)
    few = 1.2 / 3 ** 0.5
    tol = 1e-6 + gap * np.log(2.0) * 2.0 ** -23 if type_ == "f32" else ON_THE_WHOLE[type_]
    assert off(got, want) <= tol + few * 2.0 ** (gap - (34 if type_ != "f32" and sum(q) > 10 else 39))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prompt", [False, True], ids=["tokens", "prompts"])
def test_weights_of_f16_are_rounded_once(pkg, lib, cuda, dim, prompt):
    """One cell is ahead of the others, which have equal scores and equal scales, so that their weights are rounded alike: what comes out is off by that rounding, which is known, and the output's
    own; not by one of a weight's product with a scale."""
    rng, n, kv = np.random.default_rng(53), 128, 300 if prompt else 60     # (tokens: a page, so that all cells go by the same reference)
    a = Attn(pkg, lib, 53, "f16", 8, 2, dim, [n], [kv], scale=1.0)
    if not prompt:
        a.table_np, a.q_start_np, a.kv_np, a.max_q = np.repeat(a.table_np, n, 0), np.arange(n + 1, dtype=np.int32), np.full(n, kv, np.int32), 1
    shape = (len(a.pages_np), 2, 64)
    vn, vs = rng.integers(0, 16, shape + (dim,)), np.full(shape + (dim // 32,), 181.0 / 128.0)
    kn, ks, first = np.full(shape + (dim,), 8), np.zeros(shape + (dim // 32,)), a.table_np[0, 0]
    kn[first, :, 0, 0], ks[first, :, 0, 0], vs[first, :, 0] = 0, -0.125, 0.0     # a key of 1, a value of 0
    a.pages_np = R.pack(kn.astype(np.uint8), ks, vn.astype(np.uint8), vs)
    x = rng.uniform(0.05, 6.0, (n, 8))
    a.q.view(n, 8, dim)[..., 0] = torch.from_numpy(x).cuda().half()
    a.q_np = a.q.double().cpu().numpy()
    a.upload()
    a.call()
    got, want = result(a)
    w = 2.0 ** 15 * np.exp(-a.q_np.reshape(n, 8, dim)[..., 0])
    # not next to the middle of two f16 numbers: a score of 16 bits is a sum of up to 8 * 32 magnitudes of queries in 4 steps of 2^-23, an eighth of which it is: 1e-4 at most
    sure = np.float16(w * (1 - 1e-4)) == np.float16(w * (1 + 1e-4))
    want = want * (np.float16(w).astype(np.float64) / w)[..., None]
    assert sure.mean() > 0.5
    # sums of some hundred numbers of up to 8 * 1.5 in 32 bits: 1e-5
    beyond = np.abs(got - want) - R.HALF_STEP["f16"] * 1.001 * np.abs(want) - 2.0 ** -24 - 1e-5
    assert beyond[sure].max() <= 0.0


@pytest.mark.parametrize("type_", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q,kv,heads,kv_heads,window,first", [([1] * 8, [400 + 90 * i for i in range(8)], 16, 4, 0, 0), ([1] * 4, [5000, 700, 90, 2000], 32, 8, 0, 0),
                                                              ([4, 5, 3], [500, 320, 900], 8, 2, 200, 4), ([300], [900], 8, 2, 0, 0), ([150, 200, 1], [700, 2000, 800], 4, 2, 0, 0),
                                                              ([400], [1500], 4, 4, 300, 10)], ids=str)
def test_sixteen_bits_on_the_whole(pkg, lib, cuda, type_, dim, q, kv, heads, kv_heads, window, first):
    a = Attn(pkg, lib, 44, type_, heads, kv_heads, dim, q, kv, window, first)
    a.call()
    a.check()
    assert off(*result(a)) <= ON_THE_WHOLE[type_]


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("per", ["block", "page", "cell"])
@pytest.mark.parametrize("largest", [4.0, 21760.0])
@BOTH
def test_values_of_very_different_scales(pkg, lib, cuda, type_, dim, per, largest, q, kv):
    """Values 2^12 apart between blocks, pages or cells, up to the largest that a cache holds, and a page of zeros: each block of the output as near as if it were alone."""
    a = Attn(pkg, lib, 45, type_, 8, 2, dim, q, kv)
    rng, n = np.random.default_rng(46), len(a.pages_np)
    shape = {"block": (1, 1, 1, dim // 32, 1), "page": (n, 1, 1, dim // 32, 1), "cell": (n, 2, 64, dim // 32, 1)}[per]
    small = np.arange(dim // 32).reshape(shape) % 2 if per == "block" else rng.random(shape) < 0.5
    v = np.clip(rng.standard_normal((n, 2, 64, dim // 32, 32)), -2.5, 2.5) * (largest / 2.5) * np.where(small, 2.0 ** -12, 1.0)
    v[a.table_np[0, 1]] = 0.0
    a.pages_np = R.pack(*R.quantize(rng.standard_normal((n, 2, 64, dim))), *R.quantize(v.reshape(n, 2, 64, dim)))
    a.upload()
    a.call()
    got, want = result(a)
    for b in range(dim // 32):
        g, w = got[..., 32 * b:32 * b + 32], want[..., 32 * b:32 * b + 32]
        # f16 results below its normal range have steps of 2^-24
        assert np.linalg.norm(g - w) <= (3e-6 if type_ == "f32" else ON_THE_WHOLE[type_]) * np.linalg.norm(w) + (2.0 ** -25 * w.size ** 0.5 if type_ == "f16" else 0.0), b


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_rows_of_any_magnitude_one_by_one(pkg, lib, cuda, type_, q, kv):
    """Queries from 1e-30 to 1e5: rows whose best score leads by more than all scores' errors give that cell's value, others are near on their own."""
    a = Attn(pkg, lib, 47, type_, 8, 2, 128, q, kv)
    a.q = (a.q.double() * torch.from_numpy((10.0 ** np.linspace(-30, 5, a.tokens))[:, None]).cuda()).to(TORCH[type_])
    a.q_np = a.q.double().cpu().numpy()
    a.call()
    got, want = result(a)
    half, single = R.HALF_STEP[type_] * 1.01, 0
    for s in range(len(q)):
        k, v = (x.transpose(1, 0, 2, 3).reshape(2, -1, 128) for x in R.unpack(a.pages_np[a.table_np[s, :-(-kv[s] // 64)]], 128))
        for i in range(q[s]):
            row, see = a.q_np[a.q_start_np[s] + i].reshape(2, 4, 128), kv[s] - q[s] + i + 1
            for h in range(8):
                kk, qq = k[h // 4, :see], row[h // 4, h % 4]
                z = kk @ qq * a.scale
                mag, g, w = np.abs(kk) @ np.abs(qq) * a.scale, got[a.q_start_np[s] + i, h], want[a.q_start_np[s] + i, h]
                best = np.sort(z)[::-1]
                err = 2 * 136 * 2.0 ** -23 * mag.max()
                if see > 1 and best[0] - best[1] > 2 * err + 30.0:
                    chosen = v[h // 4, z.argmax()]
                    assert np.all(np.abs(g - chosen) <= half * np.abs(chosen) + 1e-5 * np.abs(chosen).max())
                    single += 1
                elif err < 1e-3:
                    few = 1e-5 + 2.0 ** -22 * mag.max() if type_ == "f32" else 3 * ON_THE_WHOLE[type_]      # (of 128 numbers)
                    assert np.linalg.norm(g - w) <= few * np.linalg.norm(w) + 1e-6 * (type_ != "f32")
    assert single >= (8 if sum(q) < 10 else 100)


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
@pytest.mark.parametrize("scale", [1e4, 3e5])
def test_large_scores(pkg, lib, cuda, type_, q, kv, scale):
    """Scores whose own rounding is more than a binary order: weights stay finite, and the cell that is ahead by more than all errors is what comes out, but for the roundings of a weight that is no
    power of two then and of the output."""
    a = Attn(pkg, lib, 54, type_, 8, 2, 128, q, kv, scale=scale)
    a.call()
    got, want = result(a)
    single, half = 0, R.HALF_STEP[type_] + (2.0 ** -11 if type_ != "f32" else 0.0)
    for s in range(len(q)):
        k, v = (x.transpose(1, 0, 2, 3).reshape(2, -1, 128) for x in R.unpack(a.pages_np[a.table_np[s, :-(-kv[s] // 64)]], 128))
        for i in range(q[s]):
            row, see = a.q_np[a.q_start_np[s] + i].reshape(8, 128), kv[s] - q[s] + i + 1
            for h in range(8):
                z, mag = k[h // 4, :see] @ row[h] * scale, (np.abs(k[h // 4, :see]) @ np.abs(row[h])).max() * scale
                assert mag < 2e9 and np.abs(z).max() < 4e7
                g, best = got[a.q_start_np[s] + i, h], np.sort(z)[::-1]
                assert np.all(np.abs(g) <= np.abs(v[h // 4, :see]).max(0) * (1 + 1.01 * half + 1e-5))
                if see == 1 or best[0] - best[1] > 4 * 136 * 2.0 ** -23 * mag + 30.0:
                    chosen = v[h // 4, z.argmax()]
                    assert np.all(np.abs(g - chosen) <= half * 1.01 * np.abs(chosen) + 1e-5 * np.abs(chosen).max())
                    single += 1
    assert single >= sum(q) * 4


# ---------------------------------------------------------------------------------------------------------------- long and mixed batches
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,beside", [(2130, 0), (2130, 33), (16130, 0), (16130, 33)])
def test_prompts_in_f32_behind_many_cells(pkg, lib, cuda, dim, kv, beside):
    """An error that does not grow with the length, also where items stay whole (more than 32 sequences): tensor cores cut off half a step of 2^-23 in the mean of what they add to, 32 times
    (16 cells, high and low parts) before the sum goes to one of 32 bits, and that sum grows from nothing: 2 / 3 * 32 * 2^-24 = 1.3e-6; a score is added up in 16 such steps, 0.6e-6."""
    a = Attn(pkg, lib, 48, "f32", 4, 1, dim, [130] + [1] * beside, [kv] + [0] * beside)
    a.call()
    a.check()
    assert off(*result(a)) <= (1.3e-6 ** 2 + 0.6e-6 ** 2) ** 0.5


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,kv", [(40, 500), (200, 16000)])
def test_tokens_in_f32_behind_many_cells(pkg, lib, cuda, dim, n, kv):
    """The same for single tokens (which share their pages here), where a warp has up to 225 pages of a sequence: 16 cells are added up in 4 steps that cut off, their sums in 32 bits."""
    a = Attn(pkg, lib, 52, "f32", 8, 8, dim, [n], [kv])
    a.table_np, a.q_start_np, a.kv_np, a.max_q = np.repeat(a.table_np, n, 0), np.arange(n + 1, dtype=np.int32), np.full(n, kv, np.int32), 1
    a.upload()
    a.call()
    torch.cuda.synchronize()
    k, v = (torch.from_numpy(np.ascontiguousarray(x.transpose(1, 0, 2, 3).reshape(8, -1, dim)[:, :kv])).cuda() for x in R.unpack(a.pages_np[a.table_np[0, :-(-kv // 64)]], dim))
    q = torch.from_numpy(a.q_np).cuda().view(n, 8, dim).transpose(0, 1)
    want = torch.softmax(q @ k.transpose(1, 2) * a.scale, -1) @ v
    assert off(a.out.double().view(n, 8, dim).transpose(0, 1).cpu().numpy(), want.cpu().numpy()) <= 1e-6


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [20, 40])
def test_a_prompt_beside_many_tokens(pkg, lib, cuda, type_, tokens):
    """Long items are cut with up to 32 sequences, and stay whole with more."""
    a = Attn(pkg, lib, 49, type_, 8, 2, 128, [1] * tokens + [200] + [1], [100 + 30 * i for i in range(tokens)] + [6000, 77])
    a.call()
    a.check()
    assert off(*result(a)) <= (3e-6 if type_ == "f32" else ON_THE_WHOLE[type_])


# ---------------------------------------------------------------------------------------------------------------- buffers and graphs
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@BOTH
def test_queries_and_results_in_one_buffer(pkg, lib, cuda, type_, q, kv):
    """Rows of queries with rows of results between them: ranges interleave, rows do not."""
    a = Attn(pkg, lib, 50, type_, 8, 2, 128, q, kv)
    alone = a.call(torch.full_like(a.out, 7.0))
    joint = torch.full((a.tokens, 2 * 1024 + 8), 7.0, dtype=TORCH[type_], device="cuda")
    joint[:, :1024] = a.q
    a.q, a.ldq, a.ldo, out = joint, joint.shape[1], joint.shape[1], joint[:, 1024:]
    queries = joint[:, :1024].clone()
    a.call(out)
    torch.cuda.synchronize()
    assert torch.equal(joint[:, 1024:2048], alone) and torch.equal(joint[:, :1024], queries) and bool((joint[:, 2048:] == 7.0).all())


@pytest.mark.parametrize("tokens", [5, 700])
def test_append_with_its_results_in_the_same_rows(pkg, lib, cuda, tokens):
    """Rows of queries, keys, values and turned queries: what goes out lies between what is read."""
    H, HK, D, P = 4, 2, 128, -(-tokens // 64)
    x = torch.randn(tokens, (2 * H + 2 * HK) * D, device="cuda").to(torch.bfloat16)
    before, W, e = x.clone(), x.shape[1], x.element_size()
    cells, pos = torch.arange(tokens, device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda")
    rope = pkg.RopeArgs(D, 2, 4096, 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0, None)
    got = []
    for apart in (False, True):
        pages = torch.zeros(P, HK, R.chunk_bytes(D), dtype=torch.uint8, device="cuda")
        cache, q_out = pkg.Kv4Cache(pages.data_ptr(), P, 1, HK, D), torch.zeros(tokens, H * D, dtype=torch.bfloat16, device="cuda")
        at = [C.c_void_p(x.data_ptr() + i * D * e) for i in (0, H, H + HK, H + 2 * HK)]
        lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, 30, at[0], W, ptr(q_out) if apart else at[3], H * D if apart else W, at[1], W, at[2], W, tokens, H, ptr(cells), ptr(pos), None, None,
                                         0.0, C.byref(rope), None))
        torch.cuda.synchronize()
        got.append((q_out if apart else x[:, (H + 2 * HK) * D:].clone(), pages))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and torch.equal(x[:, :(H + 2 * HK) * D], before[:, :(H + 2 * HK) * D])


FIRST_CALL = """
import sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import torch
import pkgload
from test_gpu_kv4 import Attn
pkg = pkgload.load()
lib = pkg.Lib.get()
a = Attn(pkg, lib, 51, "f32", 8, 2, 128, [1, 200], [300, 400])
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a.call()
for _ in range(2):
    a.out.fill_(7.0)
    g.replay()
    a.check()
print("as it should be")
"""


def test_first_call_of_a_process_is_captured(cuda):
    """Nothing has to be called once in front of a capture."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=str(Path(__file__).resolve().parent.parent))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as it should be" in r.stdout, r.stdout[-1000:] + r.stderr[-3000:]
