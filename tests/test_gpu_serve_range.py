"""The operators around the 4-bit cache at the ends of their ranges, against their definitions in 64 bits (ref_serve.py): temperatures, rows that are alike, tables and groups that end early."""
import ctypes as C

import numpy as np
import pytest
import torch

import ref_kv4 as R
import ref_serve as V
from gpu_util import ptr
from test_gpu_serve import TYPES, Batch, drafted, stream, verify

pytestmark = pytest.mark.gpu
LOWEST = np.finfo(np.float32).min


@pytest.fixture(autouse=True)
def weights_that_count_as_nothing(monkeypatch):
    """Weights below 2^-960 of a row's largest count as 0, where numbers of 64 bits go on to 2^-1074: at temperatures as small as here's that is what all others of a row have."""
    full = V.softmax

    def softmax(x, t):
        w = full(x, t)
        if w is None:
            return None
        w = np.where(w < 2.0 ** -960 * w.max(), 0.0, w)
        return w / w.sum()

    monkeypatch.setattr(V, "softmax", softmax)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_verification_at_any_temperature(lib, cuda, type_, with_draft, masked):
    """Every 1 / temperature from the smallest number to the largest, at largest logits of 1 to 60 000: a first draft that is the target's largest, and one that is drawn."""
    rng = np.random.default_rng(70)
    pairs = [(t, top) for t in (0.0, 1e-45, 1e-38, 1e-31, 1e-20, 1e-3, 20.0, 1e3, 1e5, 1e6, 1e7, 5e7, 1e8, 1e9, 1e10, 1e12, 1e18, 1e20, 1e30, np.finfo(np.float32).max) for top in (1.0, 24.3, 130.0, 900.0, 6e4)]
    drafts, vocab = [2] * len(pairs), 3001
    target, draft, _, u, v = drafted(rng, "f32", vocab, drafts, spread=2.5, apart=0.7)
    row = np.arange(len(u)) + np.repeat(np.arange(len(pairs)), drafts)
    tops = np.array([top for _, top in pairs])
    hold = lambda x: torch.from_numpy(x.astype(np.float32)).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[type_]).float().numpy()
    target = hold(target + (np.repeat(tops, 3) - target.max(-1))[:, None])
    draft = hold(draft + (np.repeat(tops, 2) - draft.max(-1))[:, None])
    if masked:
        target[:, 2000:2500], draft[:, 100:600] = -np.inf, -np.inf
        target[::2, 700:900], draft[::2, 800:900] = hold(np.float32([LOWEST if type_ != "f16" else -65504.0])), hold(np.float32([LOWEST if type_ != "f16" else -65504.0]))
    tokens = np.array([int(np.argmax(target[r])) if i % 2 == 0 else int(rng.integers(0, vocab)) for i, r in enumerate(row)], dtype=np.int32)
    verify(lib, type_, target, draft if with_draft else None, drafts, tokens, np.array([t for t, _ in pairs], np.float32), u, v)


@pytest.mark.parametrize("with_draft", [True, False])
def test_verification_of_the_largest_and_the_lowest_logits(lib, cuda, with_draft):
    """Rows whose largest logit is the type's lowest number, beside -inf; rows with both ends of the type, at temperatures that leave something of either."""
    rng = np.random.default_rng(71)
    drafts, vocab = [2] * 12, 2500
    target, draft, _, u, v = drafted(rng, "f32", vocab, drafts)
    for x in (target, draft):
        x[:18] = np.where(rng.random((len(x[:18]), vocab)) < 0.5, LOWEST, -np.inf)
        x[18:] = np.where(rng.random((len(x[18:]), vocab)) < 0.5, LOWEST, -LOWEST)
    tokens = np.array([int(rng.choice(np.nonzero(np.isfinite(target[i + i // 2]))[0])) for i in range(24)], dtype=np.int32)
    t = np.array([1.0, 0.7, 1e9, 1e-40, 0.0, 3e38, 1.0, 0.0, 1e-38, 3e-39, 1e9, 1e-45], np.float32)
    verify(lib, "f32", target, draft if with_draft else None, drafts, tokens, t, u * np.float32(0.9), v)


@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens_without_weight_are_not_accepted(lib, cuda, with_draft):
    """A drafted token so far below the largest logit of both models that it has no weight in either: 0 < 0 is false, whatever u."""
    rng = np.random.default_rng(72)
    drafts, vocab = [1] * 24, 4001
    target, draft, _, u, v = drafted(rng, "f32", vocab, drafts)
    tokens = rng.integers(0, vocab, 24).astype(np.int32)
    target[2 * np.arange(24), tokens], draft[np.arange(24), tokens] = -30.0, -30.0
    u[::4] = 0.0
    verify(lib, "f32", target, draft if with_draft else None, drafts, tokens, np.float32([40.0, 1e3, 1e4] * 8), u, v)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("vocab", [3, 900, 20001])
def test_rows_that_are_alike_leave_the_targets_weights(lib, cuda, type_, vocab):
    """Draft and target have equal rows, and the token cannot be accepted (none, outside of the vocabulary, masked in both): of max(p - q, 0) nothing is left, p is drawn from."""
    rng = np.random.default_rng(73)
    drafts = [1] * 48
    target, _, _, u, v = drafted(rng, type_, vocab, drafts)
    target[::6, 1] = -np.inf
    draft = target[::2].copy()
    tokens = np.array([1 if i % 3 == 0 else -1 if i % 3 == 1 else vocab + i for i in range(48)], dtype=np.int32)
    verify(lib, type_, target, draft, drafts, tokens, rng.choice([1.0, 0.7, 1.4], 48), u, v)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("case", [([2, 1], [300, 64], [1, 2, 1], [5, 70, 0], 8, 2), ([64], [4000], [1] * 64, [1 + 3 * i for i in range(64)], 8, 8), ([3, 40], [600, 3000], [70, 200, 1] + [1] * 40, [70, 300, 1] + [9] * 40, 16, 8)],
                         ids=["few", "apart", "prompts"])
def test_a_prefix_ends_with_its_table(pkg, lib, cuda, type_, case):
    """Lengths of prefixes far beyond what their tables have room for: cells are those of the pages that are there, and no more pages are walked or counted."""
    groups, prefix, q, kv, heads, kv_heads = case
    b = Batch(pkg, lib, 80, type_, heads, kv_heads, 128, q, kv, groups, prefix)
    b.prefix_np[:] = [1 << 30, (1 << 31) - 1][:len(prefix)]
    b.upload()
    b.attend()
    b.check()


@pytest.mark.parametrize("q,kv,groups,prefix", [([70, 200, 1], [70, 300, 1], [3], [600]), ([1] * 24, [9 + i for i in range(24)], [24], [6000])], ids=["prompts", "apart"])
def test_items_are_cut_by_the_pages_of_both_tables(pkg, lib, cuda, q, kv, groups, prefix):
    """A plan of cut items adds up their key tiles in 30 bits: with a table of prefixes whose rows have room for more, items stay whole, and the launch that joins pieces is not made."""
    b = Batch(pkg, lib, 81, "bf16", 16, 8, 128, q, kv, groups, prefix)
    counts = []
    for ld in (b.prefix_table_np.shape[1], 2 * (2 ** 30 // (184 * 8)), 2 ** 23):      # (the one row of the table is read as far as the prefix goes, whatever the rows' stride)
        b.out.fill_(7.0)
        b.lse.fill_(7.0)
        before = lib.c.pb200_kernel_launches()
        lib.check(lib.c.pb200_kv4_attn_shared(C.byref(b.cache), 0, R.CODE["bf16"], ptr(b.q), b.ldq, ptr(b.out), b.ldo, b.heads, len(kv), ptr(b.q_start), ptr(b.kv), ptr(b.table), b.table_np.shape[1], 1,
                                              ptr(b.group), ptr(b.prefix), ptr(b.prefix_table), ld, b.tokens, b.max_q, b.scale, ptr(b.lse), b.ldl, ptr(b.ws), b.ws.numel(), stream()))
        counts.append(lib.c.pb200_kernel_launches() - before)
        b.check()
    assert counts == [3, 2, 2]


@pytest.mark.parametrize("case", ["groups", "rows"])
def test_groups_that_end_behind_the_batch(pkg, lib, cuda, case):
    """Prefixes by themselves: groups from in front of the first sequence to behind the last one; a last sequence whose rows lie behind the arrays.  The sequences that are there have their results."""
    n = 64
    b = Batch(pkg, lib, 82, "bf16", 16, 8, 128, [1] * n, [40 + i for i in range(n)], [20, n - 20], [3000, 3500])
    b.group_np = np.array([-2, 20, n + 5], np.int32) if case == "groups" else np.array([0, 20, n + 1], np.int32)
    b.upload()
    extra = case == "rows"
    q_start, kv = (torch.from_numpy(np.append(x, y).astype(np.int32)).cuda() for x, y in ((b.q_start_np, b.tokens + 7), (b.kv_np, 30)))
    table = torch.from_numpy(np.concatenate((b.table_np, b.table_np[:1]))).cuda()
    before = lib.c.pb200_kernel_launches()
    lib.check(lib.c.pb200_kv4_attn_shared(C.byref(b.cache), 0, R.CODE["bf16"], ptr(b.q), b.ldq, ptr(b.out), b.ldo, b.heads, n + extra, ptr(q_start), ptr(kv), ptr(table), b.table_np.shape[1], 2,
                                          ptr(b.group), ptr(b.prefix), ptr(b.prefix_table), b.prefix_table_np.shape[1], b.tokens, 1, b.scale, ptr(b.lse), b.ldl, ptr(b.ws), b.ws.numel(), stream()))
    assert lib.c.pb200_kernel_launches() - before >= 2, "the prefix has no kernel of its own"
    b.group_np = np.array([0, 20, n], np.int32)
    b.check()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("groups", [[1] * 64, [1] * 8, [2, 1, 1, 2, 1, 1], [1, 3] * 10], ids=lambda g: f"{len(g)}of{max(g)}")
def test_prefixes_of_few_sequences_are_walked(pkg, lib, cuda, type_, groups):
    """Long prefixes of a sequence or three each: by themselves they would save nothing.  What is walked has the bits of sequences with all pages in one table."""
    n, front = sum(groups), 16128 if len(groups) <= 8 else 4032
    b = Batch(pkg, lib, 83, type_, 16, 8, 128, [1] * n, [1 + 11 * i for i in range(n)], groups, [front] + [64] * (len(groups) - 1))
    b.prefix_np[:], b.prefix_table_np[:] = front, b.prefix_table_np[:1]                 # (groups of their own, whose pages happen to be the same)
    b.upload()
    got = b.attend().clone()
    row = np.repeat(np.arange(len(groups)), groups)
    b.table_np = np.concatenate((b.prefix_table_np[row, :front // 64], b.table_np), 1)
    b.kv_np, b.group_np = b.kv_np + front, None
    b.upload()
    b.out.fill_(7.0)
    assert torch.equal(b.attend(), got)


@pytest.mark.parametrize("max_q", [1, 6])
def test_more_queries_than_there_are_do_not_change_the_way(pkg, lib, cuda, max_q):
    """Tokens behind a prefix that they walk: with a max_q beyond what there is, too."""
    b = Batch(pkg, lib, 84, "bf16", 32, 8, 128, [1] * 16, [30 + i for i in range(16)], [16], [4032])
    got = b.attend(max_q=max_q).clone()
    b.check()
    b.table_np = np.concatenate((np.repeat(b.prefix_table_np[:, :63], 16, 0), b.table_np), 1)
    b.kv_np, b.group_np = b.kv_np + 4032, None
    b.upload()
    assert torch.equal(b.attend(max_q=max_q), got)


MIXED_CASES = [
    # groups, prefix, q, heads, kv_heads: prompts in front of a group's tokens, among them and behind them, of rows that fill tiles by themselves, and drafts beside both
    ([71], [2200], [1] * 30 + [400] + [1] * 40, 16, 8), ([40, 0, 33], [2300, 100, 1500], [130] + [1] * 39 + [2] * 15 + [257, 0, 61] + [3] * 15, 16, 8), ([9] * 34, [1088] * 34, [1] * 300 + [60] + [1] * 5, 8, 8),
    ([50, 2, 1], [3200, 3200, 64], [1] * 49 + [40] + [1, 300] + [25], 8, 8),
]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", range(len(MIXED_CASES)))
def test_tokens_share_a_prefix_beside_prompts(pkg, lib, cuda, type_, dim, case):
    """Sequences of many rows walk the prefix; those of few have it read once, as in a call of their own."""
    groups, prefix, q, heads, kv_heads = MIXED_CASES[case]
    b = Batch(pkg, lib, 85, type_, heads, kv_heads, dim, q, [n + 7 * (i % 20) for i, n in enumerate(q)], groups, prefix)
    before = lib.c.pb200_kernel_launches()
    b.attend()
    assert lib.c.pb200_kernel_launches() - before >= 3, "the prefix has no kernel of its own"
    b.check()
    first = b.out.clone()
    b.out.fill_(7.0)
    b.attend(lse=False)
    assert torch.equal(b.out, first)
    if dim == 128:
        return
    most = 20
    b.out.fill_(7.0)
    b.lse.fill_(7.0)
    b.attend(max_q=most)
    b.check(most=most)


def test_graph_of_tokens_beside_prompts(pkg, lib, cuda):
    """One graph: prefixes by themselves and not, prompts that come and go, another call on the workspace between."""
    n = 60
    b = Batch(pkg, lib, 86, "bf16", 16, 8, 128, [1] * n + [150], [20 + i for i in range(n + 1)], [n + 1], [2700])
    other = Batch(pkg, lib, 87, "f32", 8, 8, 128, [100] + [1] * 40, [100] + [30] * 40, [41], [2500])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.attend()
        for prefix, q in ((2700, [1] * n + [150]), (100, [1] * n + [150]), (2699, [1] * 20 + [60] + [1] * 30 + [50] + [1] * 9), (2700, [1] * (n + 1))):
            b.prefix_np[:], b.q_start_np[:] = prefix, np.concatenate(([0], np.cumsum(q)))
            b.prefix.copy_(torch.from_numpy(b.prefix_np))
            b.q_start.copy_(torch.from_numpy(b.q_start_np))
            b.out.fill_(7.0)
            b.lse.fill_(7.0)
            graph.replay()
            b.check()
            other.attend(ws=b.ws)
        other.check()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
def test_tokens_beside_a_prompt_of_more_tiles_than_a_plan_has(pkg, lib, cuda, type_):
    """A prompt between tokens with more tiles of rows than items are cut by: the tokens have what they have without it."""
    n, long = 128, 12500
    b = Batch(pkg, lib, 88, type_, 4, 1, 128, [1] * n, [3 + i for i in range(n)], [n], [10240])
    half, rng = n // 2, np.random.default_rng(89)
    prompt = torch.from_numpy(rng.standard_normal((long, b.ldq)).astype(np.float32)).cuda().to(b.q.dtype)
    q = torch.cat((b.q[:half], prompt, b.q[half:]))
    out, lse = torch.full((n + long, b.ldo), 7.0, dtype=b.q.dtype, device="cuda"), torch.full((n + long, b.ldl), 7.0, device="cuda")
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()
    starts = np.concatenate((np.arange(half + 1), half + long + np.arange(half + 1)))
    kv = np.concatenate((b.kv_np[:half], [long], b.kv_np[half:]))
    table = np.full((n + 1, -(-long // R.CELLS)), -1)
    table[:half, :b.table_np.shape[1]], table[half + 1:, :b.table_np.shape[1]] = b.table_np[:half], b.table_np[half:]
    table[half] = np.arange(table.shape[1]) % len(b.pages_np)
    d = [dev(starts), dev(kv), dev(table), dev([0, n + 1])]
    ws = torch.zeros(lib.c.pb200_kv4_attn_shared_workspace_bytes(4, 1, 128, n + long), dtype=torch.uint8, device="cuda")
    before = lib.c.pb200_kernel_launches()
    lib.check(lib.c.pb200_kv4_attn_shared(C.byref(b.cache), 0, R.CODE[type_], ptr(q), b.ldq, ptr(out), b.ldo, 4, n + 1, ptr(d[0]), ptr(d[1]), ptr(d[2]), table.shape[1], 1, ptr(d[3]), ptr(b.prefix),
                                          ptr(b.prefix_table), b.prefix_table_np.shape[1], n + long, long, b.scale, ptr(lse), b.ldl, ptr(ws), ws.numel(), stream()))
    assert lib.c.pb200_kernel_launches() - before == 4, "the prefix has no kernel of its own"
    torch.cuda.synchronize()
    assert not torch.any(torch.all(out == 7.0, 1))
    b.out.copy_(torch.cat((out[:half], out[half + long:])))
    b.lse.copy_(torch.cat((lse[:half], lse[half + long:])))
    b.check()
