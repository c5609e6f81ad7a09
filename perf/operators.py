"""Operators over a cache of 4-bit keys and values in pages: what a program that serves models from such a cache calls, token by token and prompt by
prompt, through the C ABI.

  append    ``pb200_kv4_append``: queries and keys normed per head and rotated, keys and values to their cells as 4-bit rows (and ``pb200_kv4_load``,
            which gives the values back that the cells stand for)
  attend    ``pb200_kv4_attn``: attention of a ragged batch, single tokens and prompts, over the pages of its sequences; all cells up to the query's own, or
            a window of them and the first few
  copy      ``pb200_kv4_copy_pages``: whole pages, all layers, for a sequence that forks
  compact   ``pb200_kv4_compact``: the cells of a sequence that are kept, to pages of their own, for a cache that evicts

The cache.  A page holds 64 cells, each a key row and a value row of ``dim`` numbers per layer and head; per layer and head a page is a chunk of
``64 * dim / 2`` bytes of keys, as many of values, and 64 * dim / 32 scales (float16) of each.  A number is ``(n - 8) * scale``, n its 4 bits and the
scale that of its block of 32 numbers, with 8 significant bits (so that each number is a float16 exactly):

  scale of a block    the number of largest magnitude (of several, the first) / -8, rounded to 8 significant bits, then to float16
  n                   round(x / scale) + 8, at most 15 (8 where the scale is 0); NaN counts as 0, magnitudes beyond 21760 as 21760

Where bits lie, for cell t (of 64), number d, block b = d / 32 of NB = dim / 32:

  keys      row t of dim / 2 bytes; 32-bit word (d / 8 % 4) * NB + b; of its 8 numbers, number e at bit 4 * (e / 2) + 16 * (e % 2)
  values    row r = t - t % 8 + t % 8 / 2 + 4 * (t % 2); 16-bit word (g ^ (4 * (r / 2 % 2))) * NB + b with g = d / 4 % 8; number d % 4 at bit 4 * (d % 4)
  scales    entry (t / 2 * NB + b) * 2 + t % 2
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False      # False: plain forms; True: the framework's operators
DEV = "cuda"
CELLS = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 30}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one generated token of one request behind a context of a thousand, a layer of an 8B model: the smallest call, one per layer and token
        {"name": "attend_token_1000", "kind": "attend", "type": "f32", "heads": 32, "kv_heads": 8, "dim": 128, "q": "1", "kv": "1001", "window": 0, "first": 0},
        # 32 requests that decode together, contexts of all lengths up to 8192
        {"name": "attend_batch_32", "kind": "attend", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "1*32", "kv": "17..8192", "window": 0, "first": 0},
        # two documents of a hundred thousand tokens, a layer of a 70B model: what a 4-bit cache is for
        {"name": "attend_long_2", "kind": "attend", "type": "bf16", "heads": 64, "kv_heads": 8, "dim": 128, "q": "1*2", "kv": "131071,65001", "window": 0, "first": 0},
        # endless conversations: a window of 1024 cells and the first four, heads of 64
        {"name": "attend_window_16", "kind": "attend", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 64, "q": "1*16", "kv": "900..16384", "window": 1024, "first": 4},
        # the prompt of one request from the start, a layer of an 8B model
        {"name": "attend_prompt_2048", "kind": "attend", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "2048", "kv": "2048", "window": 0, "first": 0},
        # prompts in pieces behind what is there already, and a request that decodes beside them, in 32 bits
        {"name": "attend_ragged_f32", "kind": "attend", "type": "f32", "heads": 16, "kv_heads": 4, "dim": 128, "q": "700,300,77,1", "kv": "2700,300,5077,4097", "window": 0, "first": 0},
        # the rows of that prompt into the cache, queries and keys normed and rotated
        {"name": "append_prompt_2048", "kind": "append", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 2048, "norm": True, "rot": 128, "mode": 2, "far": 0},
        # the tokens of a batch of 64 at far positions, rotated in neighbouring pairs
        {"name": "append_batch_64", "kind": "append", "type": "f32", "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 64, "norm": False, "rot": 128, "mode": 0, "far": 100000},
        # the last page of a sequence that forks, a small model
        {"name": "copy_pages_2", "kind": "copy", "layers": 4, "kv_heads": 4, "dim": 64, "pages": 64, "count": 2},
        # the pages of 16 beams, 32 layers of an 8B model
        {"name": "copy_pages_48", "kind": "copy", "layers": 32, "kv_heads": 8, "dim": 128, "pages": 128, "count": 48},
        # one long request gives up half of its cells
        {"name": "compact_8000", "kind": "compact", "layers": 8, "kv_heads": 8, "dim": 128, "kv": "8000", "keep": 0.5},
        # a batch whose drafts were accepted in part
        {"name": "compact_batch_6", "kind": "compact", "layers": 2, "kv_heads": 4, "dim": 64, "kv": "300,64,65,511,1,130", "keep": 0.8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["token", "token", "token", "prompt", "prompt", "append", "copy", "compact"])
    dim, kv_heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8])
    if kind == "token":
        group = rng.choice([1, 2, 3, 4, 7, 8, 16])
        n = _log_int(rng, 1, 64)
        most = _log_int(rng, 1, min(100000, max(2, 200000 * 8 // (n * kv_heads))))
        q = rng.choice([1, 1, 1, 2, 5])
        return {"kind": "attend", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "q": "%d*%d" % (q, n),
                "kv": "%d..%d" % (max(1, most // rng.choice([1, 3, 50])), max(q, most)), "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), "first": rng.choice([0, 4, 65])}
    if kind == "prompt":
        group, kv_heads = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4])
        q = [_log_int(rng, 2, 1500) for _ in range(rng.choice([1, 1, 2, 4]))]
        more = [rng.choice([0, 0, _log_int(rng, 1, 2500)]) for _ in q]
        while group * kv_heads * sum(n * (n + 2 * m) for n, m in zip(q, more)) > 1 << 27:
            q = [(n + 1) // 2 for n in q]
        kv = [n + m for n, m in zip(q, more)]
        return {"kind": "attend", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "q": ",".join(map(str, q)),
                "kv": ",".join(map(str, kv)), "window": rng.choice([0, 0, _log_int(rng, 1, 2048)]), "first": rng.choice([0, 1, 70])}
    if kind == "append":
        rot = rng.choice([0, dim // 2, dim, dim])
        return {"kind": "append", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * rng.choice([1, 4, 5]), "kv_heads": kv_heads, "dim": dim, "tokens": _log_int(rng, 1, 2048),
                "norm": rng.random() < 0.5, "rot": rot, "mode": rng.choice([0, 2]), "far": rng.choice([0, rng.randrange(1, 200000)])}
    if kind == "copy":
        layers, pages = _log_int(rng, 1, 32), rng.randrange(16, 100)
        return {"kind": "copy", "layers": layers, "kv_heads": kv_heads, "dim": dim, "pages": pages, "count": rng.randrange(1, pages // 2 - 2)}
    kv = [_log_int(rng, 1, 2000) for _ in range(rng.randrange(1, 5))]
    return {"kind": "compact", "layers": _log_int(rng, 1, 8), "kv_heads": kv_heads, "dim": dim, "kv": ",".join(map(str, kv)), "keep": rng.choice([0.1, 0.5, 0.9, 1.0])}


def _numbers(text, n=None):
    """"3,5", "1*4" (four ones) or "3..50" (n numbers between, spread like the multiples of the golden ratio; the last one is the largest)"""
    if ".." in text:
        lo, hi = map(int, text.split(".."))
        lo = min(lo, hi)
        return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n - 1)] + [hi]
    if "*" in text:
        v, k = map(int, text.split("*"))
        return [v] * k
    return [int(v) for v in text.split(",")]


def _lengths(case):
    q = _numbers(case["q"])
    return q, _numbers(case["kv"], len(q))


# ---------------------------------------------------------------------------------------------------------------- the cache's format, in elementary operations
def _quantize(x):
    """float32 [..., dim] -> (4 bits each as uint8 [..., dim], scales float16 [..., dim / 32])"""
    b = torch.where(torch.isnan(x), 0.0, x).clamp(-21760.0, 21760.0).reshape(*x.shape[:-1], -1, 32)
    first = b.abs().argmax(-1, keepdim=True)
    scale = (b.gather(-1, first) / -8.0).to(torch.bfloat16).to(torch.float16)
    s = scale.float()
    n = torch.where(s == 0, 8.0, torch.round(b / torch.where(s == 0, 1.0, s)) + 8.0).clamp(0.0, 15.0)
    return n.to(torch.uint8).reshape(x.shape), scale.squeeze(-1)


def _pack_k(n):
    """[..., dim] 4 bits each -> bytes [..., dim / 2] of a key row"""
    x = n.reshape(*n.shape[:-1], -1, 4, 2, 2, 2)                # b, c, z, nibble, o: number 4 z + 2 nibble + o of a word
    x = x.movedim((-4, -5, -1, -3, -2), (-5, -4, -3, -2, -1))   # c, b, o, z, nibble
    return (x[..., 0] | x[..., 1] << 4).reshape(*n.shape[:-1], -1)


def _unpack_k(raw):
    x = raw.reshape(*raw.shape[:-1], 4, -1, 2, 2)               # c, b, o, z
    x = torch.stack((x & 15, x >> 4), -1)                       # c, b, o, z, nibble
    x = x.movedim((-4, -5, -2, -1, -3), (-5, -4, -3, -2, -1))   # b, c, z, nibble, o
    return x.reshape(*raw.shape[:-1], -1)


def _turn(x):
    """value rows of 8 cells [..., 8 rows, 8 words, NB] with the words of rows 2, 3, 6 and 7 in the order of the others, and back"""
    y = x.reshape(*x.shape[:-3], 2, 2, 2, 2, 4, x.shape[-1])    # row: (odd cell, second half, -), word: (half, -)
    return torch.stack((y[..., 0, :, :, :, :], y[..., 1, :, :, :, :].flip(-3)), -5).reshape(x.shape)


def _pack_v(n):
    """[..., 64, dim] 4 bits each -> bytes [..., 64, dim / 2] of the value rows of a page"""
    x = n.reshape(*n.shape[:-1], -1, 8, 4).transpose(-2, -3)    # cells, g, b, number
    w = (x[..., 0::2] | x[..., 1::2] << 4)                      # cells, g, b, byte
    w = w.reshape(*n.shape[:-2], 8, 4, 2, 8, -1).transpose(-3, -4)    # eights, odd cell, pair, g, (b, byte)
    return _turn(w.reshape(*n.shape[:-2], 8, 8, 8, -1)).reshape(*n.shape[:-1], -1)


def _rows_v(raw):
    """bytes [..., 64, dim / 2] of a page's value rows -> the same by cell, words in their order: [..., 64, 8, bytes of a word]"""
    w = _turn(raw.reshape(*raw.shape[:-2], 8, 8, 8, -1))
    return w.reshape(*raw.shape[:-2], 8, 2, 4, 8, w.shape[-1]).transpose(-3, -4).reshape(*raw.shape[:-1], 8, -1)


def _rows_v_back(w):
    x = w.reshape(*w.shape[:-3], 8, 4, 2, 8, w.shape[-1]).transpose(-3, -4).reshape(*w.shape[:-3], 8, 8, 8, -1)
    return _turn(x).reshape(*w.shape[:-2], -1)


def _unpack_v(raw):
    w = _rows_v(raw)
    w = w.reshape(*w.shape[:-1], -1, 2)                         # cells, g, b, byte
    x = torch.stack((w & 15, w >> 4), -1).flatten(-2)           # cells, g, b, number
    return x.transpose(-2, -3).reshape(*raw.shape[:-1], -1)


def _scales(raw, dim):
    """bytes of a page's scales [..., 64 * dim / 16] -> float16 [..., 64, dim / 32]"""
    x = raw.contiguous().view(torch.float16).reshape(*raw.shape[:-1], 32, dim // 32, 2)
    return x.transpose(-1, -2).reshape(*raw.shape[:-1], 64, dim // 32)


def _scales_back(s):
    x = s.reshape(*s.shape[:-2], 32, 2, s.shape[-1]).transpose(-1, -2).contiguous()
    return x.reshape(*s.shape[:-2], -1).view(torch.uint8)


def _parts(dim):
    rows, sc = CELLS * dim // 2, CELLS * dim // 16
    return (0, rows), (rows, 2 * rows), (2 * rows, 2 * rows + sc), (2 * rows + sc, 2 * rows + 2 * sc)


def _chunk(dim):
    return _parts(dim)[3][1]


def _page_bytes(k, v):
    """float32 [..., 64, dim] each -> chunks [..., bytes]"""
    kn, ks = _quantize(k)
    vn, vs = _quantize(v)
    return torch.cat((_pack_k(kn).flatten(-2), _pack_v(vn).flatten(-2), _scales_back(ks), _scales_back(vs)), -1)


def _page_values(raw, dim):
    """chunks [..., bytes] -> keys and values float32 [..., 64, dim]"""
    kr, vr, ks, vs = (raw[..., a:b] for a, b in _parts(dim))
    k = _unpack_k(kr.reshape(*raw.shape[:-1], CELLS, dim // 2)).float() - 8.0
    v = _unpack_v(vr.reshape(*raw.shape[:-1], CELLS, dim // 2)).float() - 8.0
    return k * _scales(ks, dim).float().repeat_interleave(32, -1), v * _scales(vs, dim).float().repeat_interleave(32, -1)


# ---------------------------------------------------------------------------------------------------------------- random inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(0xCAC4E + 7919 * int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _fill(g, pages, dim):
    """keys with a few strong channels, as rotated keys have them, and values; a few pages at a time"""
    n, layers, heads = pages.shape[:3]
    strong = 1.0 + 4.0 * (torch.rand(layers, heads, 1, dim, generator=g, device=DEV) > 0.97)
    step = max(1, (1 << 25) // (layers * heads * CELLS * dim))
    for i in range(0, n, step):
        m = min(step, n - i)
        pages[i:i + m] = _page_bytes(_randn(g, m, layers, heads, CELLS, dim) * strong, _randn(g, m, layers, heads, CELLS, dim))


def _tables(g, lens, extra):
    """pages of the sequences in a mixed order out of a pool with `extra` more: (table int32 [n, most], pool size); -1 behind a sequence's last page"""
    need = [-(-n // CELLS) for n in lens]
    pool = sum(need) + extra
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    ends = torch.tensor([0] + need, device=DEV).cumsum(0)
    col = torch.arange(max(max(need), 1), device=DEV)
    at = ends[:-1, None] + col
    return torch.where(at < ends[1:, None], order[at.clamp(max=pool - 1)], -1).to(torch.int32).contiguous(), pool


class _State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    g = _gen(seed)
    S = _State(case=case, kind=case["kind"])
    dim, hk = case["dim"], case["kv_heads"]
    if case["kind"] == "attend":
        q, kv = _lengths(case)
        S.update(n_seq=len(q), max_q=max(q), max_kv=max(kv), tokens=sum(q))
        table, pool = _tables(g, kv, 3)
        pages = torch.empty(pool, 1, hk, _chunk(dim), dtype=torch.uint8, device=DEV)
        _fill(g, pages, dim)
        ends = np.concatenate(([0], np.cumsum(q)))
        S.update(pages=pages, table=table, q_start=torch.from_numpy(ends.astype(np.int32)).to(DEV), kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV),
                 q=_randn(g, S["tokens"], case["heads"], dim).to(TYPES[case["type"]]),
                 place=torch.from_numpy(np.concatenate([np.arange(n) + i * max(q) for i, n in enumerate(q)])).to(DEV))
        S["out"] = torch.zeros_like(S["q"])
        S["ws"] = torch.zeros(_workspace(), dtype=torch.uint8, device=DEV)
    elif case["kind"] == "append":
        t, h = case["tokens"], case["heads"]
        pool = -(-t // CELLS) + 3
        pages = torch.zeros(pool, 1, hk, _chunk(dim), dtype=torch.uint8, device=DEV)
        _fill(g, pages, dim)
        cells = torch.randperm(pool, generator=g, device=DEV)[torch.arange(t, device=DEV) // CELLS] * CELLS + torch.arange(t, device=DEV) % CELLS
        if case["far"]:     # one token each of many sequences
            cells = torch.randperm(pool * CELLS, generator=g, device=DEV)[:t]
            pos = torch.randint(0, case["far"], (t,), generator=g, device=DEV)
        else:
            pos = torch.arange(t, device=DEV)
        S.update(pages=pages, cells=cells.contiguous(), pos=pos.to(torch.int32), qkv=_randn(g, t, (h + 2 * hk) * dim).to(TYPES[case["type"]]),
                 qw=1.0 + 0.1 * _randn(g, dim), kw=1.0 + 0.1 * _randn(g, dim), eps=1e-6, base=500000.0)
        S["q_out"] = torch.empty(t, h, dim, dtype=TYPES[case["type"]], device=DEV)
        S["k_val"], S["v_val"] = (torch.empty(t, hk, dim, dtype=torch.float16, device=DEV) for _ in range(2))
    elif case["kind"] == "copy":
        pages = torch.empty(case["pages"], case["layers"], hk, _chunk(dim), dtype=torch.uint8, device=DEV)
        _fill(g, pages[:4], dim)
        pages[4:] = torch.randint(0, 256, (case["pages"] - 4, 1, 1, 1), generator=g, device=DEV, dtype=torch.uint8) ^ pages[torch.arange(4, case["pages"], device=DEV) % 4]
        order = np.random.RandomState(int(seed) % (1 << 31)).permutation(case["pages"]).astype(np.int32)
        n = case["count"]
        dst, src = order[:n].copy(), order[n:][np.arange(n) // 3 % (case["pages"] - n)].copy()   # three forks of each
        S.update(pages=pages, src=src, dst=dst, src_t=torch.from_numpy(src).to(DEV).long(), dst_t=torch.from_numpy(dst).to(DEV).long())
    else:
        kv = _numbers(case["kv"])
        count = [max(0, min(n, int(round(n * case["keep"])))) for n in kv]
        both, pool = _tables(g, kv + [max(c, 1) for c in count], 2)
        pages = torch.empty(pool, case["layers"], hk, _chunk(dim), dtype=torch.uint8, device=DEV)
        _fill(g, pages, dim)
        rows = [torch.randperm(n, generator=g, device=DEV)[:c].sort().values for n, c in zip(kv, count)]
        index = torch.zeros(len(kv), max(max(count), 1), dtype=torch.int32, device=DEV)
        for i, r in enumerate(rows):
            index[i, :r.numel()] = r.to(torch.int32)
        S.update(pages=pages, n_seq=len(kv), table=both[:len(kv)].contiguous(), to=both[len(kv):].contiguous(), index=index, count=torch.tensor(count, dtype=torch.int32, device=DEV),
                 most=max(max(count), 1))
        S["to_seq"], S["to_col"] = (S.to >= 0).nonzero(as_tuple=True)     # the pages that the sequences have
        S["to_pages"] = S.to[S.to_seq, S.to_col].long()
    return S


def _workspace():
    """bytes of the attention's workspace, which a program allocates once, zeroed"""
    return 64 << 20


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _visible(S, cells):
    """[n_seq, max_q, cells]: which cells a query sees"""
    c = S.case
    n_q = (S.q_start[1:] - S.q_start[:-1])[:, None, None]
    p = S.kv_len[:, None, None] - n_q + torch.arange(S.max_q, device=DEV)[None, :, None]
    i = torch.arange(cells, device=DEV)[None, None, :]
    see = i <= p
    if c["window"]:
        see = see & ((p - i < c["window"]) | (i < c["first"]))
    return see


def _plain_attend(S):
    c = S.case
    dim, hk, grp, n = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"], S.n_seq
    raw = S.pages[S.table.clamp(min=0).long(), 0]                                         # n, pages, heads, bytes
    k, v = (x.transpose(1, 2).reshape(n, hk, -1, dim) for x in _page_values(raw, dim))    # n, heads, cells, dim
    q = torch.zeros(n * S.max_q, c["heads"], dim, device=DEV)
    q[S.place] = S.q.float()
    q = q.reshape(n, S.max_q, hk, grp, dim).permute(0, 2, 1, 3, 4).reshape(n, hk, S.max_q * grp, dim)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    see = _visible(S, k.shape[2])[:, None, :, None, :].expand(n, 1, S.max_q, grp, -1).reshape(n, 1, S.max_q * grp, -1)
    s = torch.where(see, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.reshape(n, hk, S.max_q, grp, dim).permute(0, 2, 1, 3, 4).reshape(n * S.max_q, c["heads"], dim)
    return o[S.place].to(S.q.dtype)


def _angles(S, dim):
    """cosine and sine float32 [tokens, pairs], the angles in 64 bits"""
    n = S.case["rot"]
    w = torch.pow(torch.tensor(S.base, dtype=torch.float64, device=DEV), -2.0 * torch.arange(n // 2, device=DEV, dtype=torch.float64) / n)
    a = S.pos.double()[:, None] * w
    return torch.cos(a).float(), torch.sin(a).float()


def _normed(x, w, eps):
    """float32; the mean in 64 bits: a number next to a border of the 4-bit steps falls to the same side whatever the order of a sum"""
    r = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + torch.tensor(eps, dtype=torch.float32, device=DEV).double())
    return x * r.float() * w


def _rotated(x, cos, sin, n, mode):
    cos, sin = cos[:, None], sin[:, None]
    if n == 0:
        return x
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if mode == 0 else (x[..., :n // 2], x[..., n // 2:n])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if mode == 0 else torch.cat(y, -1)
    return torch.cat((y, x[..., n:]), -1)


def _plain_append(S):
    c = S.case
    dim, hk, h = c["dim"], c["kv_heads"], c["heads"]
    x = S.qkv.reshape(-1, h + 2 * hk, dim).float()
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    if c["norm"]:
        q, k = _normed(q, S.qw, S.eps), _normed(k, S.kw, S.eps)
    cos, sin = _angles(S, dim)
    q, k = _rotated(q, cos, sin, c["rot"], c["mode"]), _rotated(k, cos, sin, c["rot"], c["mode"])
    (kn, ks), (vn, vs) = _quantize(k), _quantize(v)
    page, cell = S.cells // CELLS, S.cells % CELLS
    (k0, _), (v0, _), (ks0, _), (vs0, _) = _parts(dim)
    b = torch.arange(dim // 2, device=DEV)
    heads = torch.arange(hk, device=DEV)[None, :, None]
    S.pages[page[:, None, None], 0, heads, k0 + cell[:, None, None] * (dim // 2) + b] = _pack_k(kn)
    g, nb = b // (dim // 16), dim // 32                               # 16-bit words of a value row: 8 groups of NB
    row = (cell - cell % 8 + cell % 8 // 2 + 4 * (cell % 2))[:, None]
    at = (g[None] ^ (4 * (row // 2 % 2))) * (dim // 16) + b % (dim // 16) + row * (dim // 2)
    w = vn.reshape(-1, hk, nb, 8, 4).transpose(-2, -3)
    S.pages[page[:, None, None], 0, heads, v0 + at[:, None, :]] = (w[..., 0::2] | w[..., 1::2] << 4).flatten(2)
    entry = ((cell[:, None] // 2 * nb + torch.arange(nb, device=DEV)) * 2 + cell[:, None] % 2) * 2
    entry = torch.stack((entry, entry + 1), -1).flatten(1)[:, None, :]
    S.pages[page[:, None, None], 0, heads, ks0 + entry] = ks.contiguous().view(torch.uint8)
    S.pages[page[:, None, None], 0, heads, vs0 + entry] = vs.contiguous().view(torch.uint8)
    k_val = (kn.float() - 8.0) * ks.float().repeat_interleave(32, -1)
    v_val = (vn.float() - 8.0) * vs.float().repeat_interleave(32, -1)
    return [q.to(S.qkv.dtype), k_val.half(), v_val.half(), S.pages]


def _plain_copy(S):
    S.pages[S.dst_t] = S.pages[S.src_t]
    return S.pages


def _plain_compact(S):
    c = S.case
    dim = c["dim"]
    parts = _parts(dim)

    def by_cell(raw):       # n, pages, layers, heads, bytes -> n, cells, layers, heads, bytes of a cell
        kr, vr, ks, vs = (raw[..., a:b] for a, b in parts)
        k = kr.reshape(*raw.shape[:-1], CELLS, -1)
        v = _rows_v(vr.reshape(*raw.shape[:-1], CELLS, -1)).flatten(-2)
        s = [_scales(x, dim).contiguous().view(torch.uint8) for x in (ks, vs)]
        return torch.cat((k, v, *s), -1).movedim(-2, 2).flatten(1, 2)

    old, new = by_cell(S.pages[S.table.clamp(min=0).long()]), by_cell(S.pages[S.to.clamp(min=0).long()])
    i = torch.arange(new.shape[1], device=DEV)[None]
    take = torch.zeros(S.n_seq, new.shape[1], dtype=torch.long, device=DEV)
    take[:, :S.most] = S.index.long()
    got = old[torch.arange(S.n_seq, device=DEV)[:, None], take]
    new = torch.where((i < S.count[:, None])[:, :, None, None, None], got, new)
    new = new.unflatten(1, (-1, CELLS)).movedim(2, -2)                  # n, pages, layers, heads, cells, bytes
    k, v, ks, vs = new.split((dim // 2, dim // 2, dim // 16, dim // 16), -1)
    raw = torch.cat((k.flatten(-2), _rows_v_back(v.reshape(*v.shape[:-1], 8, -1)).flatten(-2), *(_scales_back(x.contiguous().view(torch.float16)) for x in (ks, vs))), -1)
    S.pages[S.to_pages] = raw[S.to_seq, S.to_col]
    return S.pages


# ---------------------------------------------------------------------------------------------------------------- the framework's operators
def _p(t):
    return C.c_void_p(t.data_ptr())


def _cache(pkg, S):
    return pkg.Kv4Cache(S.pages.data_ptr(), S.pages.shape[0], S.pages.shape[1], S.pages.shape[2], S.case["dim"])


def _own(S):
    import pkgload
    pkg = pkgload.load()
    lib = pkg.Lib.get()
    c, cache, stream = S.case, _cache(pkg, S), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    if S.kind == "attend":
        h, dim = c["heads"], c["dim"]
        lib.check(lib.c.pb200_kv4_attn(C.byref(cache), 0, CODES[c["type"]], _p(S.q), h * dim, _p(S.out), h * dim, h, S.n_seq, _p(S.q_start), _p(S.kv_len), _p(S.table),
                                       S.table.shape[1], S.tokens, S.max_q, 1.0 / math.sqrt(dim), c["window"], c["first"], _p(S.ws), S.ws.numel(), stream), "kv4_attn")
        return S.out
    if S.kind == "append":
        h, hk, dim, t = c["heads"], c["kv_heads"], c["dim"], c["tokens"]
        ld, size, code = S.qkv.shape[1], S.qkv.element_size(), CODES[c["type"]]
        at = [C.c_void_p(S.qkv.data_ptr() + i * dim * size) for i in (0, h, h + hk)]
        rope = pkg.RopeArgs(n_dims=c["rot"], mode=c["mode"], n_ctx_orig=8192, freq_base=S.base, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0)
        lib.check(lib.c.pb200_kv4_append(C.byref(cache), 0, code, at[0], ld, _p(S.q_out), h * dim, at[1], ld, at[2], ld, t, h, _p(S.cells), _p(S.pos),
                                         _p(S.qw) if c["norm"] else None, _p(S.kw) if c["norm"] else None, S.eps, C.byref(rope), stream), "kv4_append")
        lib.check(lib.c.pb200_kv4_load(C.byref(cache), 0, CODES["f16"], _p(S.cells), t, _p(S.k_val), hk * dim, _p(S.v_val), hk * dim, stream), "kv4_load")
        return [S.q_out, S.k_val, S.v_val, S.pages]
    if S.kind == "copy":
        lib.check(lib.c.pb200_kv4_copy_pages(C.byref(cache), S.src.ctypes.data_as(C.c_void_p), S.dst.ctypes.data_as(C.c_void_p), c["count"], stream), "kv4_copy_pages")
        return S.pages
    lib.check(lib.c.pb200_kv4_compact(C.byref(cache), S.n_seq, _p(S.table), S.table.shape[1], _p(S.to), S.to.shape[1], _p(S.index), S.index.shape[1], _p(S.count), S.most, stream),
              "kv4_compact")
    return S.pages


def run(state):
    if own:
        return _own(state)
    return {"attend": _plain_attend, "append": _plain_append, "copy": _plain_copy, "compact": _plain_compact}[state.kind](state)


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def _seen(p, window, first):
    """cells that the query at position p sees"""
    if p < 0:
        return 0
    if window == 0 or p + 1 <= window:
        return p + 1
    return window + min(first, p + 1 - window)


def work(case):
    dim, hk = case["dim"], case["kv_heads"]
    row = dim // 2 + dim // 16
    size = 4 if case.get("type") == "f32" else 2
    if case["kind"] == "attend":
        q, kv = _lengths(case)
        cells = pairs = 0
        for n, length in zip(q, kv):
            p0 = length - n
            pairs += sum(_seen(p0 + i, case["window"], case["first"]) for i in range(n))
            lo = max(0, p0 - case["window"] + 1) if case["window"] else 0
            cells += length - lo + min(lo, case["first"])
        return {"bytes": 2 * sum(q) * case["heads"] * dim * size + cells * hk * 2 * row, "flops": 4 * pairs * case["heads"] * dim}
    if case["kind"] == "append":
        t, h = case["tokens"], case["heads"]
        return {"bytes": t * ((2 * h + 2 * hk) * dim * size + hk * 2 * row + 2 * hk * (row + 2 * dim) + 20), "flops": t * (h + 2 * hk) * dim * 10}
    if case["kind"] == "copy":
        src = min(-(-case["count"] // 3), case["pages"] - case["count"])
        return {"bytes": (src + case["count"]) * case["layers"] * hk * _chunk(dim), "flops": 0}
    cells = sum(max(0, min(n, int(round(n * case["keep"])))) for n in _numbers(case["kv"]))
    return {"bytes": cells * (case["layers"] * hk * 4 * row + 4), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _place(dim):
    """byte and shift of number d of cell t in a chunk, keys and values, and the byte of its scale: int64 [64, dim] each, number by number from the format's definition"""
    kb, ksh, vb, vsh, sc = (np.zeros((CELLS, dim), dtype=np.int64) for _ in range(5))
    nb, rows = dim // 32, CELLS * dim // 2
    for t in range(CELLS):
        r = t - t % 8 + t % 8 // 2 + 4 * (t % 2)
        for d in range(dim):
            b, e = d // 32, d % 8
            bit = 4 * (e // 2) + 16 * (e % 2)
            kb[t, d], ksh[t, d] = t * dim // 2 + 4 * (d // 8 % 4 * nb + b) + bit // 8, bit % 8
            bit = 4 * (d % 4)
            vb[t, d], vsh[t, d] = rows + r * dim // 2 + 2 * ((d // 4 % 8 ^ 4 * (r // 2 % 2)) * nb + b) + bit // 8, bit % 8
            sc[t, d] = 2 * rows + 2 * ((t // 2 * nb + b) * 2 + t % 2)
    return [torch.from_numpy(x).to(DEV) for x in (kb, ksh, vb, vsh, sc)]


def _value(raw, at, shift, scale):
    """float64 of the numbers at these places of chunks [n, bytes]"""
    flat = at.reshape(-1)
    n = (raw[:, flat].int() >> shift.reshape(-1).int()) & 15
    lo, hi = raw[:, scale.reshape(-1)].int(), raw[:, scale.reshape(-1) + 1].int()
    bits = lo | hi << 8
    exp, man, sign = bits >> 10 & 31, bits & 1023, 1 - 2 * (bits >> 15)
    s = torch.where(exp == 0, torch.ldexp(man.double(), torch.tensor(-24, device=DEV)), torch.ldexp(1024.0 + man.double(), exp - 25)) * sign
    return ((n - 8).double() * s).reshape(raw.shape[0], *at.shape)


def _step4(x):
    """float64 [..., dim] -> the float64 numbers that its 4 bits stand for"""
    out = torch.zeros_like(x)
    for b in range(x.shape[-1] // 32):
        y = x[..., 32 * b:32 * b + 32].clamp(-21760.0, 21760.0)
        big = torch.take_along_dim(y, y.abs().argmax(-1, keepdim=True), -1) / -8.0
        man, exp = torch.frexp(big)
        s = torch.ldexp(torch.round(man * 256.0), exp - 8)
        s = torch.where(s.abs() < 2.0 ** -14, torch.round(s * 2.0 ** 24) * 2.0 ** -24, s)
        n = torch.round(y / torch.where(s == 0, 1.0, s)).clamp(-8.0, 7.0)
        out[..., 32 * b:32 * b + 32] = torch.where(s == 0, 0.0, n * s)
    return out


def exact(case, seed):
    S = prepare(case, seed)
    dim, hk, kind = case["dim"], case["kv_heads"], case["kind"]
    if kind in ("copy", "compact"):
        return None                      # bytes that move: whole numbers
    if kind == "append":
        h = case["heads"]
        x = S.qkv.double().reshape(-1, h + 2 * hk, dim)
        parts = []
        for y, w in ((x[:, :h], S.qw), (x[:, h:h + hk], S.kw)):
            if case["norm"]:
                y = y * (y.pow(2).sum(-1, keepdim=True) / dim + float(np.float32(S.eps))).pow(-0.5) * w.double()
            y = y.clone()
            n = case["rot"]
            for i in range(n // 2):
                a, b = (2 * i, 2 * i + 1) if case["mode"] == 0 else (i, i + n // 2)
                z = torch.polar(torch.ones(len(S.pos), dtype=torch.float64, device=DEV), S.pos.double() * S.base ** (-2.0 * i / n))[:, None] * torch.complex(y[..., a], y[..., b])
                y[..., a], y[..., b] = z.real, z.imag
            parts.append(y)
        return [parts[0], _step4(parts[1]), _step4(x[:, h + hk:]), None]
    q_len, kv_len = _lengths(case)
    kb, ksh, vb, vsh, sc = _place(dim)
    grp, out, at = case["heads"] // hk, [], 0
    for s, (n, length) in enumerate(zip(q_len, kv_len)):
        np_ = -(-length // CELLS)
        o = torch.zeros(n, case["heads"], dim, dtype=torch.float64, device=DEV)
        for j in range(hk):
            raw = S.pages[S.table[s, :np_].long(), 0, j]
            ks, vs = [], []
            for i in range(0, np_, 256):
                ks.append(_value(raw[i:i + 256], kb, ksh, sc))
                vs.append(_value(raw[i:i + 256], vb, vsh, sc + CELLS * dim // 16))
            k, v = (torch.cat(z).reshape(-1, dim)[:length] for z in (ks, vs))
            cell = torch.arange(length, device=DEV)
            for i in range(0, n, 512):
                m = min(512, n - i)
                p = length - n + i + torch.arange(m, device=DEV)[:, None]
                hide = cell > p
                if case["window"]:
                    hide |= (cell <= p - case["window"]) & (cell >= case["first"])
                z = torch.einsum("thd,cd->htc", S.q[at + i:at + i + m, j * grp:(j + 1) * grp].double(), k) / math.sqrt(dim)
                z = torch.softmax(z.masked_fill(hide, -math.inf), -1).nan_to_num(0.0)
                o[i:i + m, j * grp:(j + 1) * grp] = torch.einsum("htc,cd->thd", z, v)
        out.append(o)
        at += n
    return torch.cat(out)
