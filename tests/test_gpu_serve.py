"""The operators around the 4-bit cache against their definitions in 64 bits (ref_serve.py), within bounds that follow from their roundings; whole numbers exactly."""
import ctypes as C

import numpy as np
import pytest
import torch

import ref_kv4 as R
import ref_serve as V
from gpu_util import ptr
from test_gpu_kv4 import TORCH, random_pages, rows

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def dev(x, type_=np.int32):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=type_)).cuda()


class Batch:
    """Sequences in groups with prefixes (or none), their pages in a mixed order, and the calls."""

    def __init__(self, pkg, lib, seed, type_, heads, kv_heads, dim, q, kv, groups=None, prefix=None, group_at=0, window=0, first=0, layers=1, layer=0, pad=0, front=0, behind=0, scale=None):
        rng = np.random.default_rng(seed)
        self.pkg, self.lib, self.type, self.heads, self.kv_heads, self.dim, self.window, self.first, self.layers, self.layer = pkg, lib, type_, heads, kv_heads, dim, window, first, layers, layer
        self.scale = dim ** -0.5 if scale is None else scale
        prefix = prefix or []
        lens = [max(n, 0) for n in kv + prefix]
        need = [-(-n // R.CELLS) for n in lens]
        pool = sum(need) + 2
        self.pages_np = random_pages(rng, pool, layers * kv_heads, dim)
        order, table, at = rng.permutation(pool), np.full((len(lens), max(need + [1]) + 1), -1, np.int32), 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table_np, self.prefix_table_np = table[:len(kv)], table[len(kv):]
        self.q_start_np = (front + np.concatenate(([0], np.cumsum(q)))).astype(np.int32)
        self.kv_np, self.prefix_np = np.array(kv, np.int32), np.array(prefix, np.int32)
        self.group_np = None if groups is None else (group_at + np.concatenate(([0], np.cumsum(groups)))).astype(np.int32)
        self.tokens, self.max_q = front + sum(q) + behind, max(q)
        self.ldq, self.ldo, self.ldl = heads * dim + pad, heads * dim + 2 * pad, heads + pad
        self.q, self.q_np = rows(rng, type_, self.tokens, self.ldq)
        self.out = torch.full((self.tokens, self.ldo), 7.0, dtype=TORCH[type_], device="cuda")
        self.lse = torch.full((self.tokens, self.ldl), 7.0, device="cuda")
        self.ws = torch.zeros(lib.c.pb200_kv4_attn_shared_workspace_bytes(heads, kv_heads, dim, self.tokens), dtype=torch.uint8, device="cuda")
        self.upload()

    def upload(self):
        self.pages = dev(self.pages_np, np.uint8)
        self.table, self.q_start, self.kv = dev(self.table_np), dev(self.q_start_np), dev(self.kv_np)
        if self.group_np is not None:
            self.group, self.prefix, self.prefix_table = dev(self.group_np), dev(self.prefix_np), dev(self.prefix_table_np)
        self.cache = self.pkg.Kv4Cache(self.pages.data_ptr(), len(self.pages_np), self.layers, self.kv_heads, self.dim)

    def attend(self, max_q=None, lse=True, ws=None, out=None):
        max_q, ws, out = self.max_q if max_q is None else max_q, self.ws if ws is None else ws, self.out if out is None else out
        a = [C.byref(self.cache), self.layer, R.CODE[self.type], ptr(self.q), self.ldq, ptr(out), self.ldo, self.heads, len(self.kv_np), ptr(self.q_start), ptr(self.kv), ptr(self.table),
             self.table_np.shape[1]]
        l = [ptr(self.lse) if lse else None, self.ldl, ptr(ws), ws.numel(), stream()]
        if self.group_np is None:
            self.lib.check(self.lib.c.pb200_kv4_attn_lse(*a, self.tokens, max_q, self.scale, self.window, self.first, *l), "kv4_attn_lse")
        else:
            n = len(self.group_np) - 1
            self.lib.check(self.lib.c.pb200_kv4_attn_shared(*a, n, ptr(self.group), ptr(self.prefix) if n else None, ptr(self.prefix_table) if n else None, max(1, self.prefix_table_np.shape[1]),
                                                            self.tokens, max_q, self.scale, *l), "kv4_attn_shared")
        return out

    def want(self):
        pages = self.pages_np.reshape(len(self.pages_np), self.layers, self.kv_heads, -1)[:, self.layer]
        q = self.q_np[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim)
        extra = {} if self.group_np is None else dict(group_start=self.group_np, prefix_len=self.prefix_np, prefix_table=self.prefix_table_np)
        return V.attend(q, pages, self.table_np, self.q_start_np, self.kv_np, self.kv_heads, self.dim, self.scale, self.window, self.first, **extra)

    def check(self, most=None, lse=True):
        torch.cuda.synchronize()
        assert self.lib.c.pb200_aborted() == 0
        out, got_lse = self.out.double().cpu().numpy(), self.lse.double().cpu().numpy()
        assert np.all(out[:, self.heads * self.dim:] == 7.0) and np.all(got_lse[:, self.heads:] == 7.0), "behind a row"
        out, got_lse = out[:, :self.heads * self.dim].reshape(self.tokens, self.heads, self.dim), got_lse[:, :self.heads]
        mine = np.zeros(self.tokens, bool)
        for s in range(len(self.kv_np)):
            n = self.q_start_np[s + 1] - self.q_start_np[s]
            mine[self.q_start_np[s]:self.q_start_np[s] + (n if most is None else min(n, most))] = True
        assert np.all(out[~mine] == 7.0) and np.all(got_lse[~mine] == 7.0), "rows of no sequence"
        want, bound, want_lse, lse_bound, _, _ = self.want()
        want, bound, out = want[mine], bound[mine], out[mine]
        assert np.all(np.isfinite(out))
        # two parts that become one: either within its bound, and their factors
        tol = 2 * bound + R.HALF_STEP[self.type] * np.abs(want) * 1.01
        if self.type != "f32":       # a prompt's weights are rounded to f16 (2^-11 of one at most), and what lies below its normal range is lost
            tol = tol + 2.0 ** -10 * np.abs(want).max() + 2.0 ** -20
        assert np.max(np.abs(out - want) - tol) <= 0.0, np.max(np.abs(out - want))
        if not lse:
            assert np.all(got_lse[mine] == 7.0)
            return
        got_lse, want_lse, lse_bound = got_lse[mine], want_lse[mine], lse_bound[mine]
        nothing = np.isinf(want_lse)
        assert np.all(got_lse[nothing] == -np.inf) and np.all(np.isfinite(got_lse[~nothing]))
        assert np.all(np.abs(got_lse[~nothing] - want_lse[~nothing]) <= 2 * lse_bound[~nothing])


LSE_CASES = [
    # q, kv, heads, kv_heads, window, first
    ([1], [1], 4, 4, 0, 0), ([1], [0], 8, 2, 0, 0), ([1], [700], 7, 1, 0, 0), ([1] * 5, [1, 130, 0, 64, 511], 16, 2, 0, 0), ([3], [1], 8, 2, 0, 0), ([1] * 3, [500, 64, 3], 8, 2, 100, 4),
    ([1] * 3, [20000, 9, 6400], 8, 8, 0, 0), ([17], [17], 4, 4, 0, 0), ([129], [129], 16, 2, 0, 0), ([200], [1000], 8, 2, 0, 0), ([33, 128, 1, 257], [33, 500, 900, 257], 8, 2, 0, 0),
    ([150, 400], [700, 400], 8, 2, 130, 70), ([200, 30], [100, 0], 8, 2, 0, 0), ([60], [9000], 8, 1, 0, 0),
]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", LSE_CASES, ids=lambda c: f"q{sum(c[0])}of{len(c[0])}_kv{max(c[1])}_h{c[2]}over{c[3]}_w{c[4]}_{c[5]}")
def test_logarithms(pkg, lib, cuda, type_, dim, case):
    q, kv, heads, kv_heads, window, first = case
    b = Batch(pkg, lib, 1, type_, heads, kv_heads, dim, q, kv, window=window, first=first)
    b.attend()
    b.check()


def test_logarithms_leave_the_results_of_attention_as_they_are(pkg, lib, cuda):
    for q, kv in (([1] * 9, [100 * i for i in range(9)]), ([200, 5, 70], [900, 5, 70])):
        b = Batch(pkg, lib, 2, "bf16", 16, 4, 128, q, kv)
        b.attend()
        plain = torch.full_like(b.out, 7.0)
        lib.check(lib.c.pb200_kv4_attn(C.byref(b.cache), 0, R.CODE["bf16"], ptr(b.q), b.ldq, ptr(plain), b.ldo, 16, len(kv), ptr(b.q_start), ptr(b.kv), ptr(b.table), b.table_np.shape[1], b.tokens, b.max_q,
                                       b.scale, 0, 0, ptr(b.ws), b.ws.numel(), stream()))
        assert torch.equal(plain, b.out)


SHARED_CASES = [
    # groups, prefix, q, kv, heads, kv_heads
    ([1], [1], [1], [1], 4, 4), ([2], [63], [1, 1], [1, 5], 8, 2), ([3], [64], [1] * 3, [1, 64, 65], 8, 1), ([3], [65], [1, 2, 1], [0, 2, 130], 6, 2), ([2], [0], [1, 1], [3, 0], 8, 2),
    ([8], [1000], [1] * 8, [1 + 15 * i for i in range(8)], 32, 8), ([1, 3, 2], [130, 0, 700], [1] * 6, [5, 9, 64, 1, 300, 2], 14, 2), ([4, 0, 3], [100, 50, 7], [2] * 7, [2 + 9 * i for i in range(7)], 4, 4),
    ([40], [5000], [1] * 40, [1 + 7 * i for i in range(40)], 8, 2), ([20, 30], [640, 200], [5] * 50, [5 + i for i in range(50)], 16, 4), ([1] * 35, [64 * i for i in range(35)], [1] * 35, [9] * 35, 8, 8),
    ([3], [600], [70, 200, 1], [70, 300, 1], 8, 2), ([2, 2], [500, 129], [300, 20, 33, 150], [300, 20, 100, 400], 4, 1), ([60], [3000], [1] * 60, [40] * 60, 16, 1), ([300], [257], [1] * 300, [1 + i % 70 for i in range(300)], 4, 2),
    ([2], [128], [6, 6], [2, 0], 8, 2),
]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", SHARED_CASES, ids=lambda c: f"g{'_'.join(map(str, c[0][:6]))}_p{max(c[1])}_q{sum(c[2])}_kv{max(c[3])}_h{c[4]}over{c[5]}")
def test_attention_behind_prefixes(pkg, lib, cuda, type_, dim, case):
    groups, prefix, q, kv, heads, kv_heads = case
    b = Batch(pkg, lib, 3, type_, heads, kv_heads, dim, q, kv, groups, prefix)
    b.attend()
    b.check()


# prefixes that are much work for sequences of few rows, which then are read once for all of a group's: one group, several (one of them without cells, one without sequences), more than eight, tiles of rows
# that are full, one more, and nearly empty; cells of a prefix cut into pieces or not
APART_CASES = [
    ([64], [4000], [1] * 64, [1 + 3 * i for i in range(64)], 8, 8), ([32, 0, 33, 3], [3000, 500, 2049, 0], [1] * 68, [i % 70 for i in range(68)], 16, 8), ([9] * 12, [1024 + i for i in range(12)], [1] * 108, [5] * 108, 16, 8),
    ([65], [3500], [2] * 65, [2 + i for i in range(65)], 8, 4), ([130], [640], [3, 1] * 65, [3 + i % 9 for i in range(130)], 32, 8), ([14], [20000], [4] * 14, [40] * 14, 4, 4), ([520], [500], [1] * 520, [1 + i % 5 for i in range(520)], 4, 4),
]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", APART_CASES, ids=lambda c: f"g{'_'.join(map(str, c[0][:6]))}_p{max(c[1])}_q{sum(c[2])}_kv{max(c[3])}_h{c[4]}over{c[5]}")
def test_prefixes_by_themselves(pkg, lib, cuda, type_, dim, case):
    groups, prefix, q, kv, heads, kv_heads = case
    b = Batch(pkg, lib, 60, type_, heads, kv_heads, dim, q, kv, groups, prefix)
    before = lib.c.pb200_kernel_launches()
    b.attend()
    assert lib.c.pb200_kernel_launches() - before >= 2, "the prefix has no kernel of its own"
    b.check()
    first = b.out.clone()
    b.out.fill_(7.0)
    assert torch.equal(b.attend(), first)


def test_prefixes_by_themselves_with_strides_and_rows_of_nobody(pkg, lib, cuda):
    """Sequences in front of the groups and behind them, rows around them, queries beyond the first three of a sequence, longer rows than there have to be, a layer, no logarithms."""
    n = 70
    b = Batch(pkg, lib, 61, "bf16", 16, 8, 128, [1, 2] + [1 + i % 5 for i in range(n)] + [3], [70, 3] + [5 + i for i in range(n)] + [200], [30, 40], [2000, 1777], group_at=2, layers=2, layer=1, pad=4, front=3, behind=2)
    b.attend(max_q=3)
    b.check(most=3)
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.attend(max_q=3, lse=False)
    b.check(most=3, lse=False)


def test_prefixes_by_themselves_keep_what_is_no_number_in_its_rows(pkg, lib, cuda):
    b = Batch(pkg, lib, 62, "f32", 8, 8, 128, [1] * 64, [40] * 64, [64], [3000])
    want = b.attend().clone()
    b.q[3, 5], b.q[50, 200] = float("nan"), float("inf")
    b.attend()
    torch.cuda.synchronize()
    other = [i for i in range(64) if i not in (3, 50)]
    assert torch.equal(b.out[other], want[other]) and torch.isnan(b.out[3, :128]).all() and torch.equal(b.out[3, 128:], want[3, 128:])


def test_graph_follows_prefixes_from_one_way_to_the_other(pkg, lib, cuda):
    """One graph: prefixes long enough to be by themselves, then not, then again; workspaces of other calls' sizes and other head sizes between them."""
    b = Batch(pkg, lib, 63, "f16", 16, 8, 128, [1] * 64, [50 + i for i in range(64)], [24, 40], [3000, 2500])
    small = Batch(pkg, lib, 64, "f32", 8, 8, 64, [1] * 64, [30] * 64, [64], [2000])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.attend()
        for prefix, groups in (([3000, 2500], [24, 40]), ([64, 70], [24, 40]), ([0, 2500], [1, 63]), ([2999, 0], [64, 0])):
            b.prefix_np[:], b.group_np[:] = prefix, np.concatenate(([0], np.cumsum(groups)))
            for t, x in ((b.prefix, b.prefix_np), (b.group, b.group_np)):
                t.copy_(torch.from_numpy(x))
            b.out.fill_(7.0)
            b.lse.fill_(7.0)
            graph.replay()
            b.check()
            small.out.fill_(7.0)
            small.lse.fill_(7.0)
            small.attend(ws=b.ws)
            small.check()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_sequences_outside_of_groups_strides_and_layers(pkg, lib, cuda, type_):
    """Two sequences in front of the groups and one behind; rows that are nobody's around them; rows longer than they have to be; the second of three layers."""
    b = Batch(pkg, lib, 4, type_, 8, 2, 128, [1, 3, 1, 2, 1, 40], [70, 3, 9, 130, 500, 90], [2, 1], [200, 77], group_at=2, layers=3, layer=1, pad=4, front=3, behind=2)
    b.attend()
    b.check()
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.attend(lse=False)
    b.check(lse=False)


def test_no_groups_and_negative_scale(pkg, lib, cuda):
    b = Batch(pkg, lib, 5, "f32", 8, 2, 64, [1, 3], [70, 30], [], [], scale=-0.2)
    b.attend()
    b.check()


def test_only_the_first_queries_of_a_sequence(pkg, lib, cuda):
    b = Batch(pkg, lib, 6, "f16", 8, 2, 128, [5, 2, 9], [5, 60, 90], [3], [100])
    b.attend(max_q=4)
    b.check(most=4)


def test_pages_that_are_none(pkg, lib, cuda):
    """A page number outside of the cache in a prefix's and in a sequence's table, a table that ends in front of the prefix: nobody sees these cells."""
    b = Batch(pkg, lib, 7, "f32", 8, 2, 128, [1, 2, 1], [130, 70, 5], [2, 1], [300, 64 * 7])
    b.prefix_table_np[0, 2], b.table_np[0, 1] = len(b.pages_np), 1 << 30
    b.prefix_table_np, b.prefix_np[1] = np.ascontiguousarray(b.prefix_table_np[:, :6]), 64 * 7
    b.upload()
    b.attend()
    b.check()


def test_what_nobody_sees_may_be_anything(pkg, lib, cuda):
    """Cells behind the end of a prefix and of a sequence with scales that are no numbers."""
    b = Batch(pkg, lib, 8, "bf16", 8, 2, 128, [1] * 20, [33] * 20, [20], [100])
    want = b.attend().clone()
    _, _, _, _, ks, vs = R.places(128)
    for table, length in ((b.prefix_table_np[0], 100), (b.table_np[0], 33)):
        page = b.pages_np[table[(length - 1) // 64]]
        for s in (ks, vs):
            at = s[length % 64:, ::32]
            page[:, at], page[:, at + 1] = 0, 0x7e
    b.upload()
    assert torch.equal(b.attend(), want)


def test_infinities_and_nan_in_queries_stay_in_their_rows(pkg, lib, cuda):
    b = Batch(pkg, lib, 9, "f32", 8, 2, 128, [1] * 30, [40] * 30, [30], [500])
    want = b.attend().clone()
    b.q[3, 5], b.q[17, 200] = float("nan"), float("inf")
    b.attend()
    torch.cuda.synchronize()
    other = [i for i in range(30) if i not in (3, 17)]
    assert torch.equal(b.out[other], want[other]) and torch.isnan(b.out[3, :128]).all() and torch.equal(b.out[3, 128:], want[3, 128:])


def test_equal_calls_give_equal_bits_and_share_a_workspace(pkg, lib, cuda):
    """Prefixes by either kernel, and a call without groups on the same workspace between them."""
    for q, kv, groups, prefix in (([1] * 50, [100] * 50, [50], [4000]), ([1] * 6, [100] * 6, [6], [4000]), ([100, 1, 60], [100, 30, 90], [3], [900])):
        b = Batch(pkg, lib, 10, "bf16", 16, 2, 128, q, kv, groups, prefix)
        first = b.attend().clone()
        other = Batch(pkg, lib, 11, "bf16", 16, 2, 128, [9, 1], [300, 2000])
        other.attend(ws=b.ws)
        other.check()
        for _ in range(5):
            b.out.fill_(7.0)
            assert torch.equal(b.attend(), first)


def test_graph_follows_lengths_and_groups(pkg, lib, cuda):
    b = Batch(pkg, lib, 12, "f16", 16, 4, 128, [1] * 24, [50 + i for i in range(24)], [10, 14], [700, 900])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.attend()
        for prefix, groups, kv in (([700, 900], [10, 14], None), ([640, 33], [1, 23], 7), ([0, 899], [24, 0], 40)):
            b.prefix_np[:], b.group_np[:] = prefix, np.concatenate(([0], np.cumsum(groups)))
            if kv:
                b.kv_np[:] = kv
            for t, x in ((b.prefix, b.prefix_np), (b.group, b.group_np), (b.kv, b.kv_np)):
                t.copy_(torch.from_numpy(x))
            b.out.fill_(7.0)
            b.lse.fill_(7.0)
            graph.replay()
            b.check()


def test_two_streams_with_workspaces_of_their_own(pkg, lib, cuda):
    batches = [Batch(pkg, lib, 13 + i, "bf16", 16, 4, 128, [1] * 30, [60 + i] * 30, [30], [2000 + i]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(10):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                b.attend()
    torch.cuda.synchronize()
    for b in batches:
        b.check()


# ---------------------------------------------------------------------------------------------------------------- weights of cells
def weigh(b, lse, decay, old, sums, max_q=None):
    b.lib.check(b.lib.c.pb200_kv4_weigh(C.byref(b.cache), b.layer, R.CODE[b.type], ptr(b.q), b.ldq, b.heads, len(b.kv_np), ptr(b.q_start), ptr(b.kv), ptr(b.table), b.table_np.shape[1], b.tokens,
                                        b.max_q if max_q is None else max_q, b.scale, b.window, b.first, ptr(lse), lse.shape[1], decay, ptr(old) if old is not None else None,
                                        old.shape[1] if old is not None else 0, ptr(sums), sums.shape[1], stream()), "kv4_weigh")
    torch.cuda.synchronize()


def check_weights(b, sums_before, got, decay, old, width=None):
    want, bound = b.want()[4:]
    for s, length in enumerate(max(int(x), 0) for x in b.kv_np):
        n = min(length, got.shape[1])
        assert np.array_equal(got[s, n:], sums_before[s, n:]), "behind the sequence"
        if n == 0:
            continue
        past = decay * old[s, :n] if old is not None else np.zeros(n)
        worst = np.abs(got[s, :n] - (want[s][:n] + past)) - bound[s][:n] - 2.0 ** -23 * (np.abs(past) + np.abs(want[s][:n]))
        assert worst.max() <= 0.0, (s, int(worst.argmax()), worst.max())


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", LSE_CASES + [([1] * 70, [3 * i for i in range(70)], 4, 1, 0, 0), ([1] * 600, [1 + i % 5 for i in range(600)], 2, 1, 0, 0), ([300], [300], 6, 2, 1, 0), ([9] * 3, [900, 256, 257], 12, 3, 0, 0),
                                              # more rows than a cluster holds; more kv heads than warps; a kv head whose rows are cut between CTAs; three kv heads
                                              ([600, 20], [900, 300], 16, 2, 0, 0), ([2, 1], [300, 77], 40, 20, 0, 0), ([90], [400], 16, 1, 0, 0), ([130, 7], [500, 90], 12, 3, 70, 5)],
                         ids=lambda c: f"q{sum(c[0])}of{len(c[0])}_kv{max(c[1])}_h{c[2]}over{c[3]}_w{c[4]}_{c[5]}")
def test_weights(pkg, lib, cuda, type_, dim, case):
    q, kv, heads, kv_heads, window, first = case
    b = Batch(pkg, lib, 20, type_, heads, kv_heads, dim, q, kv, window=window, first=first)
    lse = dev(np.nan_to_num(b.want()[2], nan=7.0, neginf=-np.inf), np.float32)
    rng = np.random.default_rng(1)
    width = max(max(kv), 1) + 3
    old = dev(rng.random((len(q), width)) * 3, np.float32)
    sums = torch.full((len(q), width), 5.0, device="cuda")
    weigh(b, lse, 0.75, old, sums)
    check_weights(b, np.full((len(q), width), 5.0), sums.double().cpu().numpy(), 0.75, old.double().cpu().numpy())


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("case", [(12, 9, 3000, 4, 1), (6, 9, 3000, 4, 1), (1, 9, 200, 4, 1), (6, 9, 3000, 8, 2), (40, 9, 200, 8, 2), (1, 9, 200, 8, 2), (40, 9, 200, 12, 3), (8, 9, 500, 12, 3), (1, 9, 200, 12, 3),
                                  (4, 20, 900, 12, 3), (8, 20, 200, 12, 3), (1, 20, 200, 12, 3)], ids=lambda c: "%dx%dof%d_h%dover%d" % c)
@pytest.mark.parametrize("window", [0, 90])
def test_weights_of_many_rows_however_items_are_cut(pkg, lib, cuda, type_, case, window):
    """sizes for which one, two, four or eight CTAs have an item, and one, two or four warps the same cells"""
    n, q, kv, heads, kv_heads = case
    kv = [max(0, kv - 41 * i % kv) if i else kv for i in range(n)]
    b = Batch(pkg, lib, 27, type_, heads, kv_heads, 64 if window else 128, [q] * n, kv, window=window, first=5 if window else 0)
    lse = dev(np.nan_to_num(b.want()[2], nan=7.0, neginf=-np.inf), np.float32)
    width = max(kv) + 3
    sums = torch.full((n, width), 5.0, device="cuda")
    weigh(b, lse, 0.0, None, sums)
    check_weights(b, np.full((n, width), 5.0), sums.double().cpu().numpy(), 0.0, None)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_of_many_rows_eight_bytes_apart(pkg, lib, cuda, type_, dim):
    """rows that lie on 8 bytes, but not on 16, in 16 bits; rows in front and behind that are nobody's"""
    b = Batch(pkg, lib, 28, type_, 16, 2, dim, [40, 9], [300, 170], pad=4, front=3, behind=2)
    lse = dev(np.nan_to_num(b.want()[2], nan=7.0, neginf=-np.inf), np.float32)
    sums = torch.full((2, 301), 5.0, device="cuda")
    weigh(b, lse, 0.0, None, sums)
    check_weights(b, np.full((2, 301), 5.0), sums.double().cpu().numpy(), 0.0, None)


def test_weights_behind_attention_sum_up_to_the_queries(pkg, lib, cuda):
    """attn_lse, then weigh in place twice: all weights of a row are 1, whatever kernel its logarithm came from."""
    b = Batch(pkg, lib, 21, "bf16", 16, 2, 128, [1, 80, 5], [900, 333, 64])
    b.attend()
    sums = torch.zeros(3, 1000, device="cuda")
    for k in range(1, 3):
        weigh(b, b.lse, 1.0, sums, sums)
        total = sums.double().sum(1).cpu().numpy()
        # a score's error is the same in both; what is left is the logarithm's rounding and the sums'
        assert np.abs(total / (k * 16 * np.array([1.0, 80.0, 5.0])) - 1.0).max() < 1e-5


def test_weights_of_few_sums_no_old_and_odd_strides(pkg, lib, cuda):
    """Sums of the first cells alone; no earlier sums; a decay of 0, which reads none (they are no numbers); rows longer than they have to be."""
    b = Batch(pkg, lib, 22, "f32", 8, 2, 128, [2, 1], [700, 300], layers=2, layer=1, pad=4, front=1, behind=1)
    b.attend()
    for old, decay in ((None, 3.0), (torch.full((2, 500), float("nan"), device="cuda"), 0.0)):
        sums = torch.full((2, 401), 5.0, device="cuda")
        weigh(b, b.lse, decay, old, sums)
        check_weights(b, np.full((2, 401), 5.0), sums.double().cpu().numpy(), 0.0, None)


def test_weights_of_the_last_queries_alone(pkg, lib, cuda):
    """The observation window of a prompt: q_start names its last rows, positions follow."""
    b = Batch(pkg, lib, 23, "f16", 8, 4, 64, [200], [1000])
    b.attend()
    full = b.want()[2]
    b.q_start_np = np.array([180, 200], np.int32)
    b.upload()
    sums = torch.zeros(1, 1000, device="cuda")
    weigh(b, b.lse, 1.0, None, sums)
    assert np.abs(full[180:] - b.want()[2][180:]).max() == 0.0
    check_weights(b, np.zeros((1, 1000)), sums.double().cpu().numpy(), 0.0, None)


def test_weights_of_sequences_without_queries_fade(pkg, lib, cuda):
    b = Batch(pkg, lib, 24, "bf16", 8, 2, 128, [1, 0, 2], [70, 80, 90])
    b.attend()
    old = torch.rand(3, 90, device="cuda")
    sums = torch.zeros(3, 90, device="cuda")
    weigh(b, b.lse, 0.5, old, sums)
    assert torch.equal(sums[1, :80], old[1, :80] * 0.5) and torch.all(sums[1, 80:] == 0)
    b.q_start_np[:] = [5, 2, -1, 9]                                       # in no order: nobody's
    b.upload()
    weigh(b, b.lse, 0.5, old, sums)
    assert torch.equal(sums[2, :90], old[2, :90] * 0.5)


def test_weights_of_cells_that_are_none_and_of_garbage(pkg, lib, cuda):
    b = Batch(pkg, lib, 25, "f32", 8, 2, 128, [3], [400])
    b.table_np[0, 2] = -5
    page = b.pages_np[b.table_np[0, 6]]                                   # cells 384 ..: 400 and on are nobody's
    at = R.places(128)[4][16:, ::32]
    page[:, at], page[:, at + 1] = 0, 0x7e
    b.upload()
    lse = dev(b.want()[2], np.float32)
    sums = torch.full((1, 448), 5.0, device="cuda")
    weigh(b, lse, 0.0, None, sums)
    got = sums.double().cpu().numpy()
    check_weights(b, np.full((1, 448), 5.0), got, 0.0, None)
    assert np.all(got[0, 128:192] == 0.0)


def test_weights_are_the_same_each_time_and_in_a_graph(pkg, lib, cuda):
    b = Batch(pkg, lib, 26, "bf16", 32, 8, 128, [1] * 20 + [90], [100 * i for i in range(1, 22)])
    b.attend()
    first = torch.zeros(21, 2100, device="cuda")
    weigh(b, b.lse, 1.0, None, first)
    sums = torch.zeros_like(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            b.lib.check(b.lib.c.pb200_kv4_weigh(C.byref(b.cache), 0, R.CODE["bf16"], ptr(b.q), b.ldq, 32, 21, ptr(b.q_start), ptr(b.kv), ptr(b.table), b.table_np.shape[1], b.tokens, b.max_q, b.scale, 0, 0,
                                                ptr(b.lse), b.lse.shape[1], 1.0, None, 0, ptr(sums), 2100, stream()))
        for _ in range(5):
            sums.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(sums, first)


# ---------------------------------------------------------------------------------------------------------------- which cells stay
def select(lib, sums, kv, budget, first, last, ld_index=None, max_len=None, with_kept=True):
    n, most = sums.shape[0], max(1, max(budget)) if ld_index is None else ld_index
    x = torch.from_numpy(sums).cuda()
    index, count = torch.full((n, most), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7, dtype=torch.int32, device="cuda")
    kept = torch.full((n, most + 2), -7.0, device="cuda")
    lens, budgets = dev(kv), dev(budget)
    lib.check(lib.c.pb200_kv4_select(n, ptr(x), sums.shape[1], ptr(lens), sums.shape[1] if max_len is None else max_len, ptr(budgets), first, last, ptr(index), most, ptr(count),
                                     ptr(kept) if with_kept else None, most + 2, stream()), "kv4_select")
    torch.cuda.synchronize()
    index, count, kept = index.cpu().numpy(), count.cpu().numpy(), kept.cpu().numpy()
    for s in range(n):
        length = max(0, min(kv[s], sums.shape[1], sums.shape[1] if max_len is None else max_len))
        want = V.select(sums[s], length, min(budget[s], most), first, last)
        assert count[s] == len(want) and np.array_equal(index[s, :len(want)], want), s
        assert np.all(index[s, len(want):] == -7)
        if with_kept:
            assert np.array_equal(kept[s, :len(want)], sums[s, want], equal_nan=True) and np.all(kept[s, len(want):] == -7.0)
        else:
            assert np.all(kept[s] == -7.0)


@pytest.mark.parametrize("kv,budget,first,last", [
    ([1], [1], 0, 0), ([1], [0], 0, 0), ([0], [5], 1, 1), ([5], [3], 0, 0), ([5], [3], 1, 1), ([5], [3], 2, 2), ([5], [3], 5, 5), ([5], [9], 2, 1), ([-3, 4], [2, 2], 0, 0), ([4, 4], [-1, 3], 0, 1),
    ([100, 1000, 513], [50, 100, 512], 4, 16), ([3000, 2048, 2049], [700, 1, 2048], 4, 0), ([5000, 70, 4096], [2500, 64, 4095], 0, 64), ([20000, 8193, 9000], [5000, 8192, 3], 4, 256),
    ([100003, 3, 50000], [25000, 2, 49999], 1, 1000), ([131072], [131071], 0, 0)])
@pytest.mark.parametrize("kind", ["weights", "ties", "all equal", "signs"])
def test_selection(lib, cuda, kv, budget, first, last, kind):
    rng = np.random.default_rng(30)
    x = rng.random((len(kv), max(max(kv), 1) + 3)).astype(np.float32)
    if kind == "weights":
        x = np.where(rng.random(x.shape) < 0.1, 0.0, x ** 8 * 40).astype(np.float32)
    elif kind == "ties":
        x = np.floor(x * 7).astype(np.float32)
    elif kind == "all equal":
        x[:] = 0.25
    else:
        x = ((x - 0.5) * 10.0 ** rng.integers(-40, 39, x.shape)).astype(np.float32)
        x[rng.random(x.shape) < 0.05], x[rng.random(x.shape) < 0.05], x[rng.random(x.shape) < 0.05] = np.nan, np.inf, -np.inf
        x[rng.random(x.shape) < 0.1], x[rng.random(x.shape) < 0.1] = 0.0, -0.0
    select(lib, x, kv, budget, first, last)


def test_selection_of_more_than_shared_memory_holds(lib, cuda):
    rng = np.random.default_rng(31)
    select(lib, rng.random((2, 500001)).astype(np.float32), [500001, 399999], [100000, 399998], 4, 100)


def test_selection_is_bounded_by_its_arrays(lib, cuda):
    x = np.random.default_rng(32).random((3, 900)).astype(np.float32)
    select(lib, x, [900, 2000, 300], [500, 500, 500], 4, 8, ld_index=200)
    select(lib, x, [900, 2000, 300], [500, 500, 500], 4, 8, max_len=400)
    select(lib, x, [900, 2000, 300], [100, 500, 20], 4, 8, max_len=400, with_kept=False)


# ---------------------------------------------------------------------------------------------------------------- verification
def verify(lib, type_, target, draft, drafts, tokens, t, u, v, ld_out=None, pad=0, ws=None):
    """target, draft: float32 arrays that the type holds"""
    n, total, vocab = len(drafts), sum(drafts), target.shape[1]
    start = np.concatenate(([0], np.cumsum(drafts)))

    def logits(x):
        return torch.nn.functional.pad(torch.from_numpy(x), (0, pad), value=99.0).to(TORCH[type_]).cuda() if x is not None else None

    x, y = logits(target), logits(draft)
    most = max(drafts) + 1 if ld_out is None else ld_out
    out, accepted, kv_out = torch.full((n, most), -7, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    kv = np.arange(n) * 10 + 100
    ws = torch.zeros(max(16, lib.c.pb200_verify_drafts_workspace_bytes(total)), dtype=torch.uint8, device="cuda") if ws is None else ws
    d = [dev(start), dev(tokens), dev(t, np.float32) if t is not None else None, dev(u, np.float32), dev(v, np.float32), dev(kv)]
    lib.check(lib.c.pb200_verify_drafts(R.CODE[type_], ptr(x), vocab + pad, ptr(y) if y is not None and total else None, vocab + pad, vocab, n, ptr(d[0]), total, ptr(d[1]) if total else None,
                                        ptr(d[2]) if t is not None else None, ptr(d[3]) if total else None, ptr(d[4]), ptr(accepted), ptr(out), most, ptr(d[5]), ptr(kv_out), ptr(ws), ws.numel(), stream()),
              "verify_drafts")
    torch.cuda.synchronize()
    out, accepted, kv_out = out.cpu().numpy(), accepted.cpu().numpy(), kv_out.cpu().numpy()
    for s in range(n):
        a, b = start[s], start[s + 1]
        k, token, near = V.verify(target[a + s:b + s + 1].astype(np.float64), None if draft is None else draft[a:b].astype(np.float64), tokens[a:b], 1.0 if t is None else float(np.float32(t[s])),
                                  np.float32(u[a:b]).astype(np.float64), float(np.float32(v[s])))
        # sums of a row in 32 bits: 100 000 weights of 2^-22 each, in sums of 64 at a time, are within 1e-5 of it
        assert near > 1e-5, "the test's numbers are too near to a decision"
        assert accepted[s] == k and kv_out[s] == kv[s] - (b - a) + k, s
        row = [*tokens[a:a + k], token]
        assert list(out[s, :min(most, k + 1)]) == row[:most] and np.all(out[s, k + 1:] == -7), (s, out[s], row)


def drafted(rng, type_, vocab, drafts, spread=2.5, apart=0.7):
    total = sum(drafts)
    hold = lambda x: torch.from_numpy(x.astype(np.float32)).to(TORCH[type_]).float().numpy()
    target = hold(rng.standard_normal((total + len(drafts), vocab)) * spread)
    row = np.arange(total) + np.repeat(np.arange(len(drafts)), drafts)
    draft = hold(target[row] + apart * rng.standard_normal((total, vocab)))
    tokens = np.array([int(np.argmax(d + rng.gumbel(size=vocab))) for d in draft.astype(np.float64)], dtype=np.int32)
    return target, draft, tokens, rng.random(total).astype(np.float32), rng.random(len(drafts)).astype(np.float32)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("vocab,drafts", [(1, [1, 0, 2]), (2, [3, 1]), (7, [2] * 9), (1000, [0]), (1000, [0, 0, 4]), (2047, [1, 5, 3]), (2049, [4] * 5), (16384, [3, 0, 8]), (32003, [20, 1]), (151937, [2, 3])])
def test_verification(lib, cuda, type_, with_draft, vocab, drafts):
    rng = np.random.default_rng(40)
    target, draft, tokens, u, v = drafted(rng, type_, vocab, drafts)
    t = rng.choice([1.0, 0.7, 1.4, np.inf], len(drafts))
    verify(lib, type_, target, draft if with_draft else None, drafts, tokens, t, u, v)
    verify(lib, type_, target, draft if with_draft else None, drafts, tokens, None, u, v, pad=3)


def test_verification_of_many_sequences(lib, cuda):
    rng = np.random.default_rng(41)
    drafts = [int(x) for x in rng.integers(0, 4, 700)]
    target, draft, tokens, u, v = drafted(rng, "f32", 300, drafts)
    verify(lib, "f32", target, draft, drafts, tokens, None, u, v)


def test_verification_of_more_sequences_than_fill_the_gpu(lib, cuda):
    rng = np.random.default_rng(49)
    drafts = [int(x) for x in rng.integers(0, 3, 60)]
    target, draft, tokens, u, v = drafted(rng, "bf16", 20001, drafts)
    verify(lib, "bf16", target, draft, drafts, tokens, None, u, v)


def test_a_large_vocabulary(lib, cuda):
    rng = np.random.default_rng(42)
    for with_draft in (True, False):
        target, draft, tokens, u, v = drafted(rng, "f16", 600001, [2, 1], apart=3.0)
        verify(lib, "f16", target, draft if with_draft else None, [2, 1], tokens, [0.8, 1.0], u, v)


def test_a_draft_like_the_target_is_accepted(lib, cuda):
    rng = np.random.default_rng(43)
    target, _, _, u, v = drafted(rng, "f32", 5000, [4, 6])
    row = np.arange(10) + np.repeat(np.arange(2), [4, 6])
    tokens = np.array([int(np.argmax(target[r] + rng.gumbel(size=5000))) for r in row], dtype=np.int32)
    verify(lib, "f32", target, target[row].copy(), [4, 6], tokens, None, u * 0.9, v)


def test_random_numbers_at_their_ends(lib, cuda):
    rng = np.random.default_rng(44)
    target, draft, tokens, u, v = drafted(rng, "f32", 3001, [3] * 6)
    verify(lib, "f32", target, draft, [3] * 6, tokens, None, u * 0.0, np.array([0.0, 1 - 2.0 ** -24] * 3))
    verify(lib, "f32", target, None, [3] * 6, tokens, None, u * 0.0 + np.float32(0.999), np.array([0.0, 1 - 2.0 ** -24] * 3))


@pytest.mark.parametrize("with_draft", [True, False])
def test_logits_that_are_no_numbers(lib, cuda, with_draft):
    """Masked entries (-inf and the type's lowest), NaN, +inf, rows of -inf alone, tokens outside of the vocabulary, temperatures that are none."""
    rng = np.random.default_rng(45)
    drafts = [2] * 12
    target, draft, tokens, u, v = drafted(rng, "f32", 2500, drafts)
    row = np.arange(24) + np.repeat(np.arange(12), 2)
    target[row[:8], :2000] = -np.inf
    draft[4:8, 100:2400] = np.finfo(np.float32).min
    target[row[8], ::3], draft[9, ::2] = np.nan, np.nan
    target[row[10], [5, 70, 2000]] = np.inf
    draft[11, [9, 70]] = np.inf
    target[row[12]], draft[14], target[row[16] + 1] = -np.inf, -np.inf, np.nan
    tokens[18], tokens[20] = 2500, -1
    t = np.array([1.0, 0.0, np.inf, 1.0, 1.0, 0.5, 1.0, 1.0, 1.0, 1.0, -2.0, np.nan], np.float32)
    verify(lib, "f32", target, draft if with_draft else None, drafts, tokens, t, u, v)
    t[:] = np.inf
    verify(lib, "f32", target, draft if with_draft else None, drafts, tokens, t, u, v)


def test_short_rows_of_results(lib, cuda):
    rng = np.random.default_rng(46)
    target, draft, tokens, u, v = drafted(rng, "bf16", 900, [6, 2, 5])
    verify(lib, "bf16", target, draft, [6, 2, 5], tokens, None, u * 0.5, v, ld_out=2)


def test_starts_in_no_order_leave_their_sequences_alone(lib, cuda):
    """A sequence whose start lies behind its end, or outside of the drafts, gets nothing."""
    rng = np.random.default_rng(47)
    target, draft, tokens, u, v = drafted(rng, "f32", 500, [2, 2, 2])
    x, y = torch.from_numpy(target).cuda(), torch.from_numpy(draft).cuda()
    d = [dev(tokens), dev(u, np.float32), dev(v, np.float32)]
    ws = torch.zeros(lib.c.pb200_verify_drafts_workspace_bytes(6), dtype=torch.uint8, device="cuda")
    for start, bad in (([0, 2, 1, 6], [1]), ([0, 2, 4, 9], [2]), ([-3, 2, 4, 6], [0])):
        out, accepted = torch.full((3, 4), -7, dtype=torch.int32, device="cuda"), torch.full((3,), -7, dtype=torch.int32, device="cuda")
        s = dev(start)
        lib.check(lib.c.pb200_verify_drafts(0, ptr(x), 500, ptr(y), 500, 500, 3, ptr(s), 6, ptr(d[0]), None, ptr(d[1]), ptr(d[2]), ptr(accepted), ptr(out), 4, None, None, ptr(ws), ws.numel(), stream()))
        torch.cuda.synchronize()
        for i in bad:
            assert accepted[i] == -7 and torch.all(out[i] == -7)


def test_verification_in_a_graph(lib, cuda):
    rng = np.random.default_rng(48)
    drafts = [3, 1, 4]
    target, draft, tokens, u, v = drafted(rng, "f32", 4000, drafts)
    x, y, tok, uu, vv, st = torch.from_numpy(target).cuda(), torch.from_numpy(draft).cuda(), dev(tokens), dev(u, np.float32), dev(v, np.float32), dev([0, 3, 4, 8])
    ws = torch.zeros(lib.c.pb200_verify_drafts_workspace_bytes(8), dtype=torch.uint8, device="cuda")
    out, accepted = torch.full((3, 5), -7, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lib.check(lib.c.pb200_verify_drafts(0, ptr(x), 4000, ptr(y), 4000, 4000, 3, ptr(st), 8, ptr(tok), None, ptr(uu), ptr(vv), ptr(accepted), ptr(out), 5, None, None, ptr(ws), ws.numel(), stream()))
        for scale in (1.0, 0.2, 0.99):
            uu.copy_(torch.from_numpy(u * np.float32(scale)))
            graph.replay()
            side.synchronize()
            for s, (a, b) in enumerate(((0, 3), (3, 4), (4, 8))):
                k, token, _ = V.verify(target[a + s:b + s + 1], draft[a:b], tokens[a:b], 1.0, (u * np.float32(scale)).astype(np.float64)[a:b], float(v[s]))
                assert int(accepted[s]) == k and int(out[s, k]) == token


# ---------------------------------------------------------------------------------------------------------------- together
def test_a_batch_behind_a_prefix_is_verified_weighed_and_cut(pkg, lib, cuda):
    """Requests behind a common prompt: a step of drafted tokens, verification, the lengths that it leaves, weights of the cells, half of them given up, and attention over what stayed."""
    heads, kv_heads, dim, n, k, vocab = 8, 2, 128, 6, 4, 1000
    kv = [300 + 37 * i for i in range(n)]
    b = Batch(pkg, lib, 50, "bf16", heads, kv_heads, dim, [k + 1] * n, kv, [n], [500])
    b.attend()
    b.check()
    rng = np.random.default_rng(51)
    target, draft, tokens, u, v = drafted(rng, "f32", vocab, [k] * n)
    x, y, start = torch.from_numpy(target).cuda(), torch.from_numpy(draft).cuda(), dev(np.arange(n + 1) * k)
    d = [dev(tokens), dev(u, np.float32), dev(v, np.float32)]
    ws = torch.zeros(lib.c.pb200_verify_drafts_workspace_bytes(n * k), dtype=torch.uint8, device="cuda")
    accepted, out = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, k + 1, dtype=torch.int32, device="cuda")
    lib.check(lib.c.pb200_verify_drafts(0, ptr(x), vocab, ptr(y), vocab, vocab, n, ptr(start), n * k, ptr(d[0]), None, ptr(d[1]), ptr(d[2]), ptr(accepted), ptr(out), k + 1, ptr(b.kv), ptr(b.kv), ptr(ws),
                                        ws.numel(), stream()))
    want = [V.verify(target[s * (k + 1):(s + 1) * (k + 1)], draft[s * k:(s + 1) * k], tokens[s * k:(s + 1) * k], 1.0, u.astype(np.float64)[s * k:(s + 1) * k], float(v[s]))[:2] for s in range(n)]
    assert accepted.tolist() == [a for a, _ in want] and [int(out[s, a]) for s, (a, _) in enumerate(want)] == [t for _, t in want]
    b.kv_np = b.kv.cpu().numpy()
    assert b.kv_np.tolist() == [length - k + a for length, (a, _) in zip(kv, want)]
    # one token a request at the lengths that are left
    b.q_start_np, b.max_q = np.arange(n + 1, dtype=np.int32), 1
    b.upload()
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.attend()
    b.check()
    sums = torch.zeros(n, max(kv), device="cuda")
    weigh(b, b.lse, 1.0, None, sums)
    check_weights(b, np.zeros((n, max(kv))), sums.double().cpu().numpy(), 0.0, None)
    # half of the cells to pages of their own
    keep = [int(x) // 2 for x in b.kv_np]
    per = -(-max(keep) // 64)
    extra = np.zeros((n * per, *b.pages_np.shape[1:]), np.uint8)
    to_np = (len(b.pages_np) + np.arange(n * per).reshape(n, per)).astype(np.int32)
    b.pages_np = np.concatenate((b.pages_np, extra))
    b.upload()
    index, count, kept, budget, to = torch.zeros(n, max(keep), dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, max(keep), device="cuda"), dev(keep), dev(to_np)
    lib.check(lib.c.pb200_kv4_select(n, ptr(sums), sums.shape[1], ptr(b.kv), max(kv), ptr(budget), 4, 16, ptr(index), max(keep), ptr(count), ptr(kept), max(keep), stream()))
    lib.check(lib.c.pb200_kv4_compact(C.byref(b.cache), n, ptr(b.table), b.table_np.shape[1], ptr(to), per, ptr(index), max(keep), ptr(count), max(keep), stream()))
    torch.cuda.synchronize()
    for s in range(n):
        chosen = V.select(sums[s].cpu().numpy(), int(b.kv_np[s]), keep[s], 4, 16)
        assert np.array_equal(index[s, :keep[s]].cpu().numpy(), chosen)
        old = V.read(b.pages_np, b.table_np[s], int(b.kv_np[s]), dim)
        new = V.read(b.pages.cpu().numpy(), to_np[s], keep[s], dim)
        assert np.array_equal(old[0][:, chosen], new[0][:, :keep[s]]) and np.array_equal(old[1][:, chosen], new[1][:, :keep[s]])
    b.pages_np, b.table_np, b.kv_np = b.pages.cpu().numpy(), to_np, np.array(keep, np.int32)
    b.upload()
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.attend()
    b.check()
