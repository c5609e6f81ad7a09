"""The operators of the 4-bit cache against their definitions in 64 bits (ref_kv4.py): values bit for bit, attention within bounds that follow from its roundings."""
import ctypes as C

import numpy as np
import pytest
import torch

import ref_kv4 as R
from gpu_util import ptr

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rows(rng, type_, *shape):
    """random numbers that the type holds: (device tensor, the same in 64 bits)"""
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(TORCH[type_])
    return x.cuda(), x.double().numpy()


def random_pages(rng, n, heads, dim):
    x = rng.standard_normal((2, n, heads, R.CELLS, dim)) * (1.0 + 4.0 * (rng.random((1, 1, heads, 1, dim)) > 0.95))
    return R.pack(*R.quantize(x[0]), *R.quantize(x[1]))


class Attn:
    """One ragged batch: pages, tables in a mixed order, and the call."""

    def __init__(self, pkg, lib, seed, type_, heads, kv_heads, dim, q, kv, window=0, first=0, layers=1, layer=0, pad=0, front=0, behind=0, extra_cols=1, scale=None):
        rng = np.random.default_rng(seed)
        self.lib, self.type, self.heads, self.kv_heads, self.dim, self.window, self.first, self.layer = lib, type_, heads, kv_heads, dim, window, first, layer
        self.scale = dim ** -0.5 if scale is None else scale
        need = [-(-max(n, 0) // R.CELLS) for n in kv]
        pool = sum(need) + 2
        self.pages_np = random_pages(rng, pool, layers * kv_heads, dim)
        order = rng.permutation(pool)
        self.table_np = np.full((len(q), max(need + [1]) + extra_cols), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table_np[s, :n] = order[at:at + n]
            at += n
        self.q_start_np = (front + np.concatenate(([0], np.cumsum(q)))).astype(np.int32)
        self.kv_np = np.array(kv, np.int32)
        self.tokens = front + sum(q) + behind
        self.max_q = max(q)
        self.ldq, self.ldo = heads * dim + pad, heads * dim + 2 * pad
        self.q, self.q_np = rows(rng, type_, self.tokens, self.ldq)
        self.out = torch.full((self.tokens, self.ldo), 7.0, dtype=TORCH[type_], device="cuda")
        self.ws = torch.zeros(lib.c.pb200_kv4_attn_workspace_bytes(heads, kv_heads, dim), dtype=torch.uint8, device="cuda")
        self.pkg, self.layers = pkg, layers
        self.upload()

    def upload(self):
        self.pages, self.table = torch.from_numpy(self.pages_np).cuda(), torch.from_numpy(self.table_np).cuda()
        self.q_start, self.kv = torch.from_numpy(self.q_start_np).cuda(), torch.from_numpy(self.kv_np).cuda()
        self.cache = self.pkg.Kv4Cache(self.pages.data_ptr(), len(self.pages_np), self.layers, self.kv_heads, self.dim)

    def call(self, out=None, max_q=None, stream=None):
        out = self.out if out is None else out
        rc = self.lib.c.pb200_kv4_attn(C.byref(self.cache), self.layer, R.CODE[self.type], ptr(self.q), self.ldq, ptr(out), self.ldo, self.heads, len(self.kv_np), ptr(self.q_start),
                                       ptr(self.kv), ptr(self.table), self.table_np.shape[1], self.tokens, self.max_q if max_q is None else max_q, self.scale, self.window, self.first,
                                       ptr(self.ws), self.ws.numel(), C.c_void_p(torch.cuda.current_stream().cuda_stream if stream is None else stream))
        self.lib.check(rc, "kv4_attn")
        return out

    def want(self):
        pages = self.pages_np.reshape(len(self.pages_np), self.layers, self.kv_heads, -1)[:, self.layer]
        q = self.q_np[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim)
        return R.attend(q, pages, self.table_np, self.q_start_np, self.kv_np, self.kv_heads, self.dim, self.scale, self.window, self.first)

    def check(self, out=None, most=None):
        torch.cuda.synchronize()
        assert self.lib.c.pb200_aborted() == 0
        got = (self.out if out is None else out).double().cpu().numpy()
        assert np.all(got[:, self.heads * self.dim:] == 7.0), "behind a row"
        got = got[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim)
        want, bound, reach = self.want()
        mine = np.zeros(self.tokens, bool)
        for s in range(len(self.kv_np)):
            n = self.q_start_np[s + 1] - self.q_start_np[s]
            mine[self.q_start_np[s]:self.q_start_np[s] + (n if most is None else min(n, most))] = True
        assert np.all(got[~mine] == 7.0), "rows of no sequence"
        want, bound, got = want[mine], bound[mine], got[mine]
        assert np.all(np.isfinite(got))
        # 16 bits: a prompt's weights are rounded to f16 (2^-11 of a weight at most, and of the largest value then) and what lies below its normal range is lost (2^-24 of the largest weight)
        tol = bound + R.HALF_STEP[self.type] * np.abs(want) * 1.01
        if self.type != "f32":
            tol = tol + 2.0 ** -10 * np.abs(want).max() + 2.0 ** -20
        worst = np.max(np.abs(got - want) - tol) if got.size else 0.0
        assert worst <= 0.0, f"{worst} beyond the bound; largest difference {np.max(np.abs(got - want))}"
        if self.type == "f32" and got.size and np.linalg.norm(want) > 0:
            # on the whole much nearer, but for large scores: the last four roundings of one (a block's sum onto the others, the factor, the difference to the maximum) are 2^-24 of up to
            # the sum of its magnitudes each, and change its weight by as much
            assert np.linalg.norm(got - want) <= (1e-5 + 2.0 ** -22 * reach) * np.linalg.norm(want)
        return got


TOKEN_CASES = [
    # q, kv, heads, kv_heads, window, first
    ([1], [1], 4, 4, 0, 0), ([1], [63], 8, 2, 0, 0), ([1], [64], 8, 1, 0, 0), ([1], [65], 6, 2, 0, 0), ([1], [0], 8, 2, 0, 0), ([1], [700], 7, 1, 0, 0), ([1], [2500], 32, 8, 0, 0),
    ([1] * 5, [1, 130, 0, 64, 511], 16, 2, 0, 0), ([2, 1, 0, 5], [2, 300, 90, 77], 4, 1, 0, 0), ([3], [1], 8, 2, 0, 0), ([4, 2], [2, 0], 4, 2, 0, 0),
    ([1] * 3, [500, 64, 3], 8, 2, 100, 0), ([1] * 3, [500, 300, 3], 8, 2, 1, 0), ([1, 2], [900, 400], 8, 2, 64, 4), ([1] * 2, [900, 700], 16, 1, 130, 65), ([5], [400], 10, 2, 30, 1),
    ([1] * 12, [500 + 321 * i for i in range(12)], 16, 8, 0, 0), ([1] * 3, [20000, 9, 6400], 8, 8, 0, 0),   # shares of many pages, which hold the ends of several items
    ([1] * 40, list(range(0, 400, 10)), 8, 4, 0, 0), ([1], [700], 40, 2, 0, 0), ([1] * 2, [300, 20], 3, 3, 0, 0), ([1] * 300, [3 * i for i in range(300)], 4, 1, 0, 0),
]


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", TOKEN_CASES, ids=lambda c: f"q{sum(c[0])}of{len(c[0])}_kv{max(c[1])}_h{c[2]}over{c[3]}_w{c[4]}_{c[5]}")
def test_attention_of_tokens(pkg, lib, cuda, type_, dim, case):
    q, kv, heads, kv_heads, window, first = case
    a = Attn(pkg, lib, 1, type_, heads, kv_heads, dim, q, kv, window, first)
    a.call()
    a.check()


PROMPT_CASES = [
    ([17], [17], 4, 4, 0, 0), ([64], [64], 8, 2, 0, 0), ([65], [129], 4, 1, 0, 0), ([129], [129], 16, 2, 0, 0), ([300], [300], 8, 8, 0, 0), ([200], [1000], 8, 2, 0, 0),
    ([33, 128, 1, 257], [33, 500, 900, 257], 8, 2, 0, 0), ([300], [300], 6, 2, 0, 0), ([150, 40], [700, 40], 8, 2, 100, 0), ([150, 400], [700, 400], 8, 2, 130, 70),
    ([260], [260], 8, 2, 1, 0), ([200, 30], [100, 0], 8, 2, 0, 0), ([70], [70], 48, 2, 0, 0), ([400], [3000], 4, 2, 64, 200),
]


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", PROMPT_CASES, ids=lambda c: f"q{'_'.join(map(str, c[0]))}_kv{max(c[1])}_h{c[2]}over{c[3]}_w{c[4]}_{c[5]}")
def test_attention_of_prompts(pkg, lib, cuda, type_, dim, case):
    q, kv, heads, kv_heads, window, first = case
    a = Attn(pkg, lib, 2, type_, heads, kv_heads, dim, q, kv, window, first)
    a.call()
    a.check()


MIXED = [([1, 1, 1], [300, 64, 1000]), ([200, 1, 3], [400, 90, 70])]


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_rows_strides_and_layers(pkg, lib, cuda, type_, q, kv):
    """Rows in front of the first sequence and behind the last, rows with something between them, a layer in the middle."""
    a = Attn(pkg, lib, 3, type_, 8, 2, 128, q, kv, layers=3, layer=1, pad=12, front=2, behind=3)
    a.call()
    a.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_what_no_query_sees_may_be_anything(pkg, lib, cuda, dim, q, kv):
    """Cells behind a sequence's last and pages of nobody hold NaN scales; pages that are none (negative, too large) hide their cells."""
    a = Attn(pkg, lib, 4, "f32", 8, 2, dim, q, kv)
    kb, ks, vb, vs, ksc, vsc = R.places(dim)
    owned = {int(p) for p in a.table_np.ravel() if p >= 0}
    for p in range(len(a.pages_np)):
        if p not in owned:
            a.pages_np[p] = 255
    for s, n in enumerate(kv):
        page, cell = a.table_np[s, (n - 1) // 64], (n - 1) % 64 + 1
        for sc in (ksc, vsc):
            for c in range(cell, 64):
                a.pages_np[page][:, sc[c]] = 255
                a.pages_np[page][:, sc[c] + 1] = 255
    a.table_np[0, 1], a.table_np[2, 0] = -5, len(a.pages_np)
    a.upload()
    a.call()
    a.check()


@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_windows_walk_over_anything(pkg, lib, cuda, q, kv):
    """Cells between the first and the window hold NaN scales."""
    a = Attn(pkg, lib, 5, "f32", 8, 2, 128, q, kv, window=40, first=3)
    ksc, vsc = R.places(128)[4:]
    for s, n in enumerate(kv):
        for cell in range(3, n - q[s] - 40 + 1):
            for sc in (ksc, vsc):
                page = a.table_np[s, cell // 64]
                a.pages_np[page][:, sc[cell % 64]] = 255
                a.pages_np[page][:, sc[cell % 64] + 1] = 255
    a.upload()
    a.call()
    a.check()


@pytest.mark.parametrize("window,first", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (5, 2 ** 31 - 1)])
@pytest.mark.parametrize("q,kv", [([1, 3, 1], [300, 1, 0]), ([200, 60, 1], [400, 20, 70])], ids=["tokens", "prompts"])
def test_windows_as_wide_as_can_be(pkg, lib, cuda, q, kv, window, first):
    a = Attn(pkg, lib, 18, "f32", 8, 2, 64, q, kv, window=window, first=first)
    a.call()
    a.check()


@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_queries_beyond_the_most_stay(pkg, lib, cuda, q, kv):
    a = Attn(pkg, lib, 6, "f32", 8, 2, 128, [n + 2 for n in q], kv)
    a.call(max_q=2)
    a.check(most=2)


@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_table_shorter_than_the_length(pkg, lib, cuda, q, kv):
    """Cells behind the table's end are of pages that are none."""
    a = Attn(pkg, lib, 7, "f32", 8, 2, 128, q, kv)
    a.table_np = np.ascontiguousarray(a.table_np[:, :1])
    a.upload()
    a.call()
    a.check()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_starts_in_no_order(pkg, lib, cuda, type_):
    """Sequences that go backwards have no rows; 16 times the same one, whose tiles are more than a plan has room for, is the same as once."""
    a = Attn(pkg, lib, 19, type_, 8, 2, 64, [900], [1300])
    once = a.call(a.out.clone())
    a.table_np, a.q_start_np, a.kv_np = np.repeat(a.table_np, 31, 0), np.array([0, 900] * 16, np.int32), np.full(31, 1300, np.int32)
    a.upload()
    a.call()
    torch.cuda.synchronize()
    assert lib.c.pb200_aborted() == 0
    many, once = a.out.double(), once.double()
    # (items are cut in one and whole in the other: F32's joins, and 16 bits' last one)
    assert float((many - once).abs().max()) <= 2.0 ** (-6 if type_ == "bf16" else -16) * float(once.abs().max())


@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 4.0])
def test_scales(pkg, lib, cuda, q, kv, scale):
    a = Attn(pkg, lib, 8, "f32", 8, 2, 128, q, kv, scale=scale)
    a.call()
    a.check()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_large_and_small_queries(pkg, lib, cuda, type_):
    """Rows of very different magnitudes: each is scaled by its own.  The scores of the large ones pick single cells."""
    for q, kv in MIXED:
        a = Attn(pkg, lib, 9, type_, 8, 2, 128, q, kv)
        f = (10.0 ** np.linspace(-30, 5, a.tokens))[:, None]
        a.q = (a.q.double() * torch.from_numpy(f).cuda()).to(TORCH[type_])
        a.q_np = a.q.double().cpu().numpy()
        a.call()
        a.check()


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_a_query_that_is_no_number_stays_alone(pkg, lib, cuda, type_, q, kv):
    a = Attn(pkg, lib, 10, type_, 8, 2, 128, q, kv)
    a.call()
    torch.cuda.synchronize()
    clean = a.out.clone()
    a.q[1, 3 * 128 + 5] = float("nan")
    a.call()
    torch.cuda.synchronize()
    same = (a.out == clean).reshape(a.tokens, 8, 128).all(-1)
    same[1, 3] = True
    assert bool(same.all()) and bool(torch.isnan(a.out[1, 3 * 128:4 * 128]).all())


@pytest.mark.parametrize("q,kv", MIXED + [([1, 1], [9000, 17])], ids=["tokens", "prompts", "long"])
def test_equal_calls_give_equal_bits(pkg, lib, cuda, q, kv):
    a = Attn(pkg, lib, 11, "f32", 16, 4, 128, q, kv)
    first = a.call(torch.full_like(a.out, 7.0))
    for _ in range(20):
        assert torch.equal(a.call(torch.full_like(a.out, 7.0)), first)
    a.check(first)


@pytest.mark.parametrize("q,kv", MIXED, ids=["tokens", "prompts"])
def test_captured_and_replayed_as_lengths_grow(pkg, lib, cuda, q, kv):
    """A graph reads lengths, tables and queries from device memory: replays follow them.  Eager calls between replays share the workspace."""
    a = Attn(pkg, lib, 12, "f32", 8, 2, 128, q, [n + 500 for n in kv])
    full = a.kv_np.copy()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        a.call()
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        a.call(stream=torch.cuda.current_stream().cuda_stream)
    for back in (500, 123, 0):
        a.kv_np = (full - back).astype(np.int32)
        a.kv.copy_(torch.from_numpy(a.kv_np))
        torch.cuda.synchronize()
        a.out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        a.check()
        other = a.call(torch.full_like(a.out, 7.0))
        assert torch.equal(other, a.out)


def test_calls_on_two_streams(pkg, lib, cuda):
    """Each with a workspace of its own."""
    a, b = Attn(pkg, lib, 13, "f32", 32, 8, 128, [1] * 6, [3000, 70, 900, 1500, 2, 640]), Attn(pkg, lib, 14, "bf16", 16, 2, 64, [300, 1], [800, 1200])
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        a.call(stream=s.cuda_stream)
        b.call(stream=t.cuda_stream)
    torch.cuda.synchronize()
    a.check()
    b.check()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("n,prompts", [(385, 0), (1000, 0), (500, 3)])
def test_more_sequences_than_threads(pkg, lib, cuda, type_, n, prompts):
    """Single tokens of many short sequences, a few prompts among them."""
    rng = np.random.default_rng(30)
    q, kv = [1] * n, list(rng.integers(0, 140, n))
    for i in range(prompts):
        q[100 + 150 * i], kv[100 + 150 * i] = 90 + i, 300 * i + 90
    a = Attn(pkg, lib, 17, type_, 4, 2, 64, q, [int(k) for k in kv])
    a.call()
    a.check()


def test_shared_pages(pkg, lib, cuda):
    """Sequences of one prefix share its pages."""
    a = Attn(pkg, lib, 15, "f32", 8, 2, 128, [1, 1, 2], [300, 400, 200])
    a.table_np[1, :3] = a.table_np[0, :3]
    a.table_np[2, :2] = a.table_np[0, :2]
    a.upload()
    a.call()
    a.check()


def test_pages_beyond_32_bits_of_bytes(pkg, lib, cuda):
    """A pool of 5 GB: pages behind the 4th."""
    a = Attn(pkg, lib, 16, "f32", 8, 2, 128, [1, 40], [300, 200])
    page = a.pages_np[0].size
    n = 5 * (1 << 30) // page
    pool = torch.empty(n * page, dtype=torch.uint8, device="cuda")
    far = {int(p): n - 1 - i for i, p in enumerate(np.unique(a.table_np[a.table_np >= 0]))}
    for p, to in far.items():
        pool[to * page:(to + 1) * page] = torch.from_numpy(a.pages_np[p].reshape(-1)).cuda()
    a.cache = pkg.Kv4Cache(pool.data_ptr(), n, 1, 2, 128)
    a.table = torch.from_numpy(np.vectorize(lambda p: far.get(int(p), -1))(a.table_np).astype(np.int32)).cuda()
    a.call()
    a.check()


# ---------------------------------------------------------------------------------------------------------------- cells
def append(pkg, lib, rng, type_, tokens, heads, kv_heads, dim, cells, pos, norm, n_dims, mode, n_pages, pages=None, in_place=False, layers=1, layer=0, ext=0.0, factors=None, freq_scale=1.0):
    """One call over rows of a joint product's output; returns everything there is"""
    width = (heads + 2 * kv_heads) * dim + 8
    x, x_np = rows(rng, type_, tokens, width)
    x_np = x_np[:, :-8].reshape(tokens, heads + 2 * kv_heads, dim)
    if pages is None:
        pages = torch.from_numpy(random_pages(rng, n_pages, layers * kv_heads, dim)).cuda()
    before = pages.cpu().numpy()
    cache = pkg.Kv4Cache(pages.data_ptr(), n_pages, layers, kv_heads, dim)
    q_out, ldqo = (x, width) if in_place else (torch.full((tokens, max(heads, 1) * dim), 7.0, dtype=TORCH[type_], device="cuda"), max(heads, 1) * dim)
    qw, kw = (1.0 + 0.2 * rng.standard_normal((2, dim))).astype(np.float32)
    qw_d, kw_d = torch.from_numpy(qw).cuda(), torch.from_numpy(kw).cuda()
    cells_d, pos_d = torch.from_numpy(np.asarray(cells, np.int64)).cuda(), torch.from_numpy(np.asarray(pos, np.int32)).cuda()
    ff = None if factors is None else torch.from_numpy(factors).cuda()
    rope = pkg.RopeArgs(n_dims, mode, 4096, 10000.0, freq_scale, ext, 1.0, 32.0, 1.0, None if ff is None else ff.data_ptr())
    at = [C.c_void_p(x.data_ptr() + i * dim * x.element_size()) for i in (0, heads, heads + kv_heads)]
    rc = lib.c.pb200_kv4_append(C.byref(cache), layer, R.CODE[type_], at[0] if heads else None, width, ptr(q_out) if heads else None, ldqo, at[1], width, at[2], width, tokens, heads,
                                ptr(cells_d), ptr(pos_d), ptr(qw_d) if norm in ("both", "q") else None, ptr(kw_d) if norm in ("both", "k") else None, 1e-5, C.byref(rope),
                                C.c_void_p(torch.cuda.current_stream().cuda_stream))
    lib.check(rc, "kv4_append")
    torch.cuda.synchronize()
    q = q_out[:, :heads * dim].double().cpu().numpy().reshape(tokens, heads, dim) if heads else None
    return dict(x=x_np, q=q, pages=pages.cpu().numpy(), before=before, qw=qw.astype(np.float64) if norm in ("both", "q") else None,
                kw=kw.astype(np.float64) if norm in ("both", "k") else None, cache=cache, dev=pages, x_dev=x, cells=cells_d)


def key_blocks_ok(g, x):
    """Of blocks of keys x [heads][dim] in 64 bits: whether g are their numbers.  The kernel's keys are off by as much as its queries, 12 roundings of 2^-24 of a row's magnitude (below): a block's
    largest number next to the middle of two scales has either, a key next to a border of two steps (by that, and the rounding of a quotient of up to 8.03) falls to either."""
    size, blocks = np.abs(x).max(-1)[:, None, None], x.reshape(len(x), -1, 32)
    g, off = g.reshape(blocks.shape), 12 * 2.0 ** -24 * size
    most = np.abs(blocks).max(-1, keepdims=True)
    ok = np.zeros(blocks.shape[:2], bool)
    for way in (0.0, -1.0, 1.0):
        scale = R.quantize((blocks * (1.0 + way * off / np.where(most > 0, most, 1.0))).reshape(x.shape))[1][..., None]
        some = np.where(scale != 0, scale, 1.0)
        y = blocks / some
        near = np.abs(y - np.floor(y) - 0.5) <= off / np.abs(some) + 8.03 * 2.0 ** -24
        is_ = lambda n: g == np.clip(n, -8, 7) * scale   # noqa: E731, B023
        ok |= np.all(np.where(near, is_(np.floor(y)) | is_(np.floor(y) + 1), is_(np.rint(y))), -1)
    return ok


def check_append(r, type_, heads, kv_heads, dim, cells, pos, n_dims, mode, n_pages, layers=1, layer=0, w=None, mscale=1.0):
    pos = np.asarray(pos)
    w = 10000.0 ** (-2.0 * np.arange(max(n_dims // 2, 1)) / max(n_dims, 1)) if w is None else w
    k = R.append(r["x"][:, heads:heads + kv_heads], r["kw"], 1e-5, pos, w, mode, n_dims, mscale)
    v = r["x"][:, heads + kv_heads:]
    if heads:
        q = R.append(r["x"][:, :heads], r["qw"], 1e-5, pos, w, mode, n_dims, mscale)
        # a pair's two products and their sum, the norm's two, cosine and sine: seven roundings of 2^-24 of the pair's magnitude
        size = np.abs(q).max(-1, keepdims=True)
        assert np.all(np.abs(r["q"] - q) <= 8 * 2.0 ** -24 * 1.5 * size + R.HALF_STEP[type_] * np.abs(q) * 1.01 + (2.0 ** -24 if type_ == "f16" else 0.0))
    got_k, got_v = R.unpack(r["pages"].reshape(n_pages, layers, kv_heads, -1)[:, layer], dim)
    old_k, old_v = R.unpack(r["before"].reshape(n_pages, layers, kv_heads, -1)[:, layer], dim)
    for t, c in enumerate(cells):
        if c < 0 or c >= n_pages * 64:
            continue
        for got, old, x, exact in ((got_k, old_k, k[t], False), (got_v, old_v, v[t], True)):
            g = got[c // 64, :, c % 64]
            want = R.values(*R.quantize(x))
            if exact:
                assert np.array_equal(g, want)
            else:
                step = np.abs(np.repeat(R.quantize(x)[1], 32, -1))
                assert np.all(key_blocks_ok(g, x))
                assert np.all(np.abs(g - x) <= step * (1.0 + 2.0 ** -4) + 2.0 ** -24)
            old[c // 64, :, c % 64] = g
    assert np.array_equal(got_k, old_k) and np.array_equal(got_v, old_v), "cells of no token"
    full = lambda p: p.reshape(n_pages, layers, -1)   # noqa: E731
    other = [i for i in range(layers) if i != layer]
    assert np.array_equal(full(r["pages"])[:, other], full(r["before"])[:, other]), "other layers"


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("norm", ["both", "q", "k", "none"])
@pytest.mark.parametrize("n_dims,mode", [(0, 0), (64, 0), (64, 2), (32, 2), (24, 0), (56, 2), (8, 2)])
def test_append(pkg, lib, cuda, type_, dim, norm, n_dims, mode):
    rng = np.random.default_rng(21)
    tokens, heads, kv_heads, n_pages = 9, 6, 2, 4
    cells = list(rng.permutation(n_pages * 64)[:tokens])
    cells[3], cells[5] = -1, n_pages * 64
    pos = rng.integers(0, 5000, tokens)
    r = append(pkg, lib, rng, type_, tokens, heads, kv_heads, dim, cells, pos, norm, n_dims, mode, n_pages)
    check_append(r, type_, heads, kv_heads, dim, cells, pos, n_dims, mode, n_pages)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 64, 8), (200, 4, 4), (70, 5, 1), (130, 0, 3), (33, 40, 40)])
def test_append_shapes(pkg, lib, cuda, tokens, heads, kv_heads):
    rng = np.random.default_rng(22)
    n_pages = -(-tokens // 64) + 1
    cells, pos = np.arange(tokens) + 64, np.arange(tokens) + 100000
    r = append(pkg, lib, rng, "f32", tokens, heads, kv_heads, 128, cells, pos, "both", 128, 2, n_pages)
    check_append(r, "f32", heads, kv_heads, 128, cells, pos, 128, 2, n_pages)


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n_dims,mode,heads,kv_heads", [(64, 0, 8, 2), (64, 2, 5, 3), (24, 2, 0, 1), (0, 0, 17, 1)])
def test_append_of_many_tokens(pkg, lib, cuda, type_, dim, n_dims, mode, heads, kv_heads):
    rng = np.random.default_rng(30)
    tokens, n_pages = 601, 11
    cells = list(rng.permutation(n_pages * 64)[:tokens])
    cells[0], cells[300], cells[600] = -1, n_pages * 64, -5
    pos = rng.integers(0, 5000, tokens)
    r = append(pkg, lib, rng, type_, tokens, heads, kv_heads, dim, cells, pos, "both", n_dims, mode, n_pages)
    check_append(r, type_, heads, kv_heads, dim, cells, pos, n_dims, mode, n_pages)


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens", [5, 601])
def test_append_norms_of_rows_that_are_none(pkg, lib, cuda, type_, bad, tokens):
    """A number of a row that is none makes its norm none: the query's row is NaN, the key's zeros; other rows are as they would be."""
    rng = np.random.default_rng(31)
    heads, kv_heads, dim, n_pages = 4, 2, 128, -(-tokens // 64)
    x, _ = rows(rng, type_, tokens, (heads + 2 * kv_heads) * dim)
    w, cells, size = torch.ones(dim, device="cuda"), torch.arange(tokens, device="cuda"), x.element_size()
    got = []
    for at in (None, [(1, 0, 0), (1, 3, 64), (2, 1, 127), (3, 4, 2), (tokens - 1, 5, 33)]):      # token, head (4, 5: keys), number
        y = x.clone()
        for t, h, d in at or []:
            y[t, h * dim + d] = bad
        pages = torch.zeros(n_pages, kv_heads, R.chunk_bytes(dim), dtype=torch.uint8, device="cuda")
        cache, q = pkg.Kv4Cache(pages.data_ptr(), n_pages, 1, kv_heads, dim), torch.zeros(tokens, heads * dim, dtype=TORCH[type_], device="cuda")
        of = [C.c_void_p(y.data_ptr() + i * dim * size) for i in (0, heads, heads + kv_heads)]
        lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, R.CODE[type_], of[0], y.shape[1], ptr(q), heads * dim, of[1], y.shape[1], of[2], y.shape[1], tokens, heads, ptr(cells), None,
                                         ptr(w), ptr(w), 1e-6, None, None))
        torch.cuda.synchronize()
        k = R.unpack(pages.cpu().numpy(), dim)[0].transpose(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:tokens]
        got.append((q.double().cpu().numpy().reshape(tokens, heads, dim), k))
    (q0, k0), (q1, k1) = got
    for t, h, d in at:
        if h < heads:
            row = q1[t, h]
            # an infinity's own place is inf * 0, the others x * 0
            assert np.all(np.isnan(row)) if bad != bad else np.isnan(row[d]) and np.all(np.delete(row, d) == 0.0)
            q1[t, h] = q0[t, h]
        else:
            assert np.all(k1[t, h - heads] == 0.0)
            k1[t, h - heads] = k0[t, h - heads]
    assert np.array_equal(q0, q1) and np.array_equal(k0, k1)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [40, 700])
def test_append_norms_of_any_magnitude(pkg, lib, cuda, type_, tokens):
    """Squares that leave the range of 32 bits, upwards and downwards."""
    rng = np.random.default_rng(29)
    n_pages, heads, kv_heads, dim = -(-tokens // 64), 4, 2, 128
    x = rng.standard_normal((tokens, heads + 2 * kv_heads, dim)) * (10.0 ** np.linspace(-30, 30, tokens))[:, None, None]
    x_d = torch.from_numpy(x).to(TORCH[type_]).cuda().reshape(tokens, -1)
    x = x_d.double().cpu().numpy().reshape(tokens, heads + 2 * kv_heads, dim)
    pages = torch.zeros(n_pages, kv_heads, R.chunk_bytes(dim), dtype=torch.uint8, device="cuda")
    cache, width, size = pkg.Kv4Cache(pages.data_ptr(), n_pages, 1, kv_heads, dim), x_d.shape[1], x_d.element_size()
    w = torch.ones(dim, device="cuda")
    cells, q = torch.arange(tokens, device="cuda"), torch.zeros(tokens, heads * dim, dtype=TORCH[type_], device="cuda")
    at = [C.c_void_p(x_d.data_ptr() + i * dim * size) for i in (0, heads, heads + kv_heads)]
    lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, R.CODE[type_], at[0], width, ptr(q), heads * dim, at[1], width, at[2], width, tokens, heads, ptr(cells), None, ptr(w), ptr(w), 1e-12,
                                     None, None))
    torch.cuda.synchronize()
    zero = np.zeros(tokens, np.int64)
    want_q, want_k = (R.append(y, np.ones(dim), 1e-12, zero, None, 0, 0) for y in (x[:, :heads], x[:, heads:heads + kv_heads]))
    assert np.all(np.abs(q.double().cpu().numpy().reshape(want_q.shape) - want_q) <= (4 * 2.0 ** -24 + R.HALF_STEP[type_] * 1.01) * np.abs(want_q) + 1e-38)
    k = R.unpack(pages.cpu().numpy(), dim)[0].transpose(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:tokens]
    # tiny rows: a scale below f16's normal range is off by 2^-25 at most, and a number eight times as much
    step = np.abs(np.repeat(R.quantize(want_k)[1], 32, -1))
    assert np.all(np.abs(k - want_k) <= step * (1.0 + 2.0 ** -4) + 2.0 ** -22)


def test_append_in_place_and_in_a_layer(pkg, lib, cuda):
    rng = np.random.default_rng(23)
    cells, pos = np.arange(20) * 3, np.arange(20)
    r = append(pkg, lib, rng, "bf16", 20, 4, 2, 64, cells, pos, "both", 64, 2, 2, in_place=True, layers=3, layer=2)
    check_append(r, "bf16", 4, 2, 64, cells, pos, 64, 2, 2, layers=3, layer=2)
    assert np.array_equal(r["x_dev"][:, 4 * 64:-8].double().cpu().numpy().reshape(20, 4, 64), r["x"][:, 4:]), "keys and values are read only"


def test_append_with_the_ramp_and_factors(pkg, lib, cuda):
    """YaRN: pairs that turn often keep their frequency, the others are slowed down; factors divide."""
    rng = np.random.default_rng(24)
    n, freq_scale, n_ctx = 128, 0.25, 4096
    factors = (1.0 + rng.random(n // 2)).astype(np.float32)
    cells, pos = np.arange(30), rng.integers(0, 16000, 30)
    r = append(pkg, lib, rng, "f32", 30, 4, 2, 128, cells, pos, "none", n, 2, 1, ext=1.0, factors=factors, freq_scale=freq_scale)
    dims = [n * np.log(n_ctx / (b * 2 * np.pi)) / (2 * np.log(10000.0)) for b in (32.0, 1.0)]
    lo, hi = max(0, np.floor(dims[0])), min(n - 1, np.ceil(dims[1]))
    mix = 1.0 - np.clip((np.arange(n // 2) - lo) / max(0.001, hi - lo), 0.0, 1.0)
    w = 10000.0 ** (-2.0 * np.arange(n // 2) / n) * (freq_scale * (1 - mix) + mix) / factors
    check_append(r, "f32", 4, 2, 128, cells, pos, n, 2, 1, w=w, mscale=1.0 + 0.1 * np.log(1.0 / freq_scale))


def test_append_of_numbers_that_are_none(pkg, lib, cuda):
    """The cache holds numbers only: NaN as 0, infinities as the largest; the rest of a block follows its scale."""
    pages = torch.zeros(1, 1, R.chunk_bytes(64), dtype=torch.uint8, device="cuda")
    cache = pkg.Kv4Cache(pages.data_ptr(), 1, 1, 1, 64)
    x = torch.randn(2, 64, device="cuda")
    x[0, 3], x[0, 40], x[1, 0], x[1, 63] = float("nan"), float("inf"), float("-inf"), 1e30
    cells = torch.tensor([5, 6], device="cuda")
    lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, 0, None, 0, None, 0, ptr(x), 64, ptr(x), 64, 2, 0, ptr(cells), None, None, None, 0.0, None, None))
    k, v = (torch.zeros(2, 64, dtype=torch.float32, device="cuda") for _ in range(2))
    lib.check(lib.c.pb200_kv4_load(C.byref(cache), 0, 0, ptr(cells), 2, ptr(k), 64, ptr(v), 64, None))
    torch.cuda.synchronize()
    want = R.values(*R.quantize(x.double().cpu().numpy()))
    assert np.array_equal(k.double().cpu().numpy(), want) and np.array_equal(v.double().cpu().numpy(), want) and np.isfinite(want).all()


@pytest.mark.parametrize("type_", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_load(pkg, lib, cuda, type_, dim):
    rng = np.random.default_rng(25)
    pages_np = random_pages(rng, 3, 2 * 3, dim)
    pages = torch.from_numpy(pages_np).cuda()
    cache = pkg.Kv4Cache(pages.data_ptr(), 3, 2, 3, dim)
    cells = np.concatenate((rng.permutation(192)[:70], [-1, 192, 5, 5])).astype(np.int64)
    cells_d = torch.from_numpy(cells).cuda()
    k, v = (torch.full((len(cells), 3 * dim + 4), 7.0, dtype=TORCH[type_], device="cuda") for _ in range(2))
    for kk, vv in ((k, v), (k, None), (None, v)):
        lib.check(lib.c.pb200_kv4_load(C.byref(cache), 1, R.CODE[type_], ptr(cells_d), len(cells), ptr(kk) if kk is not None else None, 3 * dim + 4, ptr(vv) if vv is not None else None,
                                       3 * dim + 4, None))
    torch.cuda.synchronize()
    want = R.unpack(pages_np.reshape(3, 2, 3, -1)[:, 1], dim)
    for got, w in ((k, want[0]), (v, want[1])):
        got = got.cpu()
        assert bool((got[:, 3 * dim:] == 7.0).all())
        for i, c in enumerate(cells):
            row = got[i, :3 * dim].reshape(3, dim)
            if c < 0 or c >= 192:
                assert bool((row == 7.0).all())
            else:
                assert torch.equal(row, torch.from_numpy(w[c // 64, :, c % 64]).to(TORCH[type_]))


@pytest.mark.parametrize("layers,kv_heads,dim,n_pages,n", [(1, 1, 64, 4, 1), (3, 2, 128, 9, 4), (2, 8, 128, 700, 300), (40, 8, 128, 6, 3)])
def test_copy_pages(pkg, lib, cuda, layers, kv_heads, dim, n_pages, n):
    size = layers * kv_heads * R.chunk_bytes(dim)
    assert size == lib.c.pb200_kv4_page_bytes(layers, kv_heads, dim)
    pages = torch.randint(0, 256, (n_pages, size), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(26)
    order = rng.permutation(n_pages).astype(np.int32)
    dst, src = order[:n].copy(), order[n:][rng.integers(0, n_pages - n, n)].copy()
    want = pages.clone()
    want[torch.from_numpy(dst).long().cuda()] = pages[torch.from_numpy(src).long().cuda()]
    cache = pkg.Kv4Cache(pages.data_ptr(), n_pages, layers, kv_heads, dim)
    lib.check(lib.c.pb200_kv4_copy_pages(C.byref(cache), src.ctypes.data, dst.ctypes.data, n, None))
    src[:], dst[:] = 0, 0          # the call has taken what it needs
    torch.cuda.synchronize()
    assert torch.equal(pages, want)


@pytest.mark.parametrize("layers,kv_heads,dim", [(1, 1, 64), (2, 3, 128), (3, 2, 64)])
def test_compact(pkg, lib, cuda, layers, kv_heads, dim):
    rng = np.random.default_rng(27)
    kv, count = [300, 64, 1, 200, 130], [150, 64, 1, 0, 129]
    from_pages, to_pages = [-(-n // 64) for n in kv], [-(-max(n, 1) // 64) for n in count]
    pool = sum(from_pages) + sum(to_pages) + 1
    pages_np = random_pages(rng, pool, layers * kv_heads, dim)
    order = rng.permutation(pool).astype(np.int32)
    table, to = np.full((5, 6), -1, np.int32), np.full((5, 4), -1, np.int32)
    at = 0
    for tab, need in ((table, from_pages), (to, to_pages)):
        for s, n in enumerate(need):
            tab[s, :n] = order[at:at + n]
            at += n
    index = np.full((5, 151), 1 << 20, np.int32)
    for s, (n, c) in enumerate(zip(kv, count)):
        index[s, :c] = np.sort(rng.permutation(n)[:c])
    index[0, 7], index[0, 9] = -3, 100000        # no cells: what they would become stays as it was
    index[4, 3] = index[4, 2]                    # one cell twice
    pages = torch.from_numpy(pages_np).cuda()
    cache = pkg.Kv4Cache(pages.data_ptr(), pool, layers, kv_heads, dim)
    dev = [torch.from_numpy(x).cuda() for x in (table, to, index, np.array(count, np.int32))]
    lib.check(lib.c.pb200_kv4_compact(C.byref(cache), 5, ptr(dev[0]), 6, ptr(dev[1]), 4, ptr(dev[2]), 151, ptr(dev[3]), 150, None))
    torch.cuda.synchronize()
    got = R.unpack(pages.cpu().numpy(), dim)
    want = [x.copy() for x in R.unpack(pages_np, dim)]
    old = R.unpack(pages_np, dim)
    for s in range(5):
        for i in range(count[s]):
            c = index[s, i]
            if 0 <= c < 6 * 64 and table[s, c // 64] >= 0:
                for w, o in zip(want, old):
                    w[to[s, i // 64], :, i % 64] = o[table[s, c // 64], :, c % 64]
    assert all(np.array_equal(g, w) for g, w in zip(got, want))


def test_a_request_from_prompt_to_fork_and_eviction(pkg, lib, cuda):
    """The operators together: a prompt goes into the cache and is attended, tokens follow, the sequence forks (its last page is copied), one branch evicts half of its cells and
    goes on.  Every step against attention in 64 bits over the values that the cells stand for."""
    rng = np.random.default_rng(28)
    H, HK, D, P = 8, 2, 128, 16
    pages = torch.zeros(P, HK, R.chunk_bytes(D), dtype=torch.uint8, device="cuda")
    cache = pkg.Kv4Cache(pages.data_ptr(), P, 1, HK, D)
    ws = torch.zeros(lib.c.pb200_kv4_attn_workspace_bytes(H, HK, D), dtype=torch.uint8, device="cuda")
    rope = pkg.RopeArgs(D, 2, 4096, 10000.0, 1.0, 0.0, 1.0, 32.0, 1.0, None)

    def step(tables, lens, new):
        """every sequence appends new tokens at its end and attends"""
        n = len(tables)
        T = n * new
        x = torch.from_numpy(rng.standard_normal((T, (H + 2 * HK) * D)).astype(np.float32)).cuda()
        pos = np.concatenate([np.arange(m - new, m) for m in lens])
        cells = np.concatenate([[t[c // 64] * 64 + c % 64 for c in range(m - new, m)] for t, m in zip(tables, lens)]).astype(np.int64)
        table = np.full((n, P), -1, np.int32)
        for s, t in enumerate(tables):
            table[s, :len(t)] = t
        dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (cells, pos.astype(np.int32), table, np.arange(0, T + 1, new).astype(np.int32), np.array(lens, np.int32))]
        at = [C.c_void_p(x.data_ptr() + i * D * 4) for i in (0, H, H + HK)]
        W = (H + 2 * HK) * D
        out = torch.full((T, H * D), 7.0, device="cuda")
        lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, 0, at[0], W, at[0], W, at[1], W, at[2], W, T, H, ptr(dev[0]), ptr(dev[1]), None, None, 0.0, C.byref(rope), None))
        lib.check(lib.c.pb200_kv4_attn(C.byref(cache), 0, 0, at[0], W, ptr(out), H * D, H, n, ptr(dev[3]), ptr(dev[4]), ptr(dev[2]), P, T, new, D ** -0.5, 0, 0, ptr(ws), ws.numel(), None))
        torch.cuda.synchronize()
        q = x[:, :H * D].double().cpu().numpy().reshape(T, H, D)
        want, bound, _ = R.attend(q, pages.cpu().numpy(), table, np.arange(0, T + 1, new), np.array(lens), HK, D, D ** -0.5)
        got = out.double().cpu().numpy().reshape(T, H, D)
        assert np.all(np.abs(got - want) <= bound + 2.0 ** -24 * np.abs(want))
        k, v = (torch.zeros(T, HK * D, device="cuda") for _ in range(2))
        lib.check(lib.c.pb200_kv4_load(C.byref(cache), 0, 0, ptr(dev[0]), T, ptr(k), HK * D, ptr(v), HK * D, None))
        torch.cuda.synchronize()
        assert np.array_equal(v.double().cpu().numpy().reshape(T, HK, D), R.values(*R.quantize(x[:, (H + HK) * D:].double().cpu().numpy().reshape(T, HK, D))))

    a = [3, 7, 1, 12]
    step([a], [200], 200)
    for i in range(3):
        step([a], [201 + i], 1)
    b = a[:3] + [5]                                # 203 cells: three full pages are shared, the fourth is copied
    src, dst = np.array([12], np.int32), np.array([5], np.int32)
    lib.check(lib.c.pb200_kv4_copy_pages(C.byref(cache), src.ctypes.data, dst.ctypes.data, 1, None))
    for i in range(4):
        step([a, b], [204 + i, 204 + i], 1)
    keep = np.sort(rng.permutation(207)[:100]).astype(np.int32)[None]
    c = [9, 0]
    dev = [torch.from_numpy(x).cuda() for x in (np.array([b], np.int32), np.array([c], np.int32), keep, np.array([100], np.int32))]
    lib.check(lib.c.pb200_kv4_compact(C.byref(cache), 1, ptr(dev[0]), 4, ptr(dev[1]), 2, ptr(dev[2]), 100, ptr(dev[3]), 100, None))
    for i in range(3):
        step([a, c], [208 + i, 101 + i], 1)
