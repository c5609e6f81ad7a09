"""Operators around a cache of 4-bit keys and values in pages that a program calls which serves many requests at once: requests behind one common prefix, requests that give up the cells
that matter least, requests whose next tokens were drafted by a smaller model.  All through the C ABI.

  shared    ``pb200_kv4_attn_shared``: attention of a ragged batch whose sequences come in groups with a prefix in common, read once for the group
  weigh     ``pb200_kv4_attn_lse`` and ``pb200_kv4_weigh``: attention with the logarithms of its sums, and from these what each cell's weights add up to over queries and heads,
            on top of what earlier calls left
  select    ``pb200_kv4_select``: which cells a sequence keeps: the first few, the last few, and of the others those with the largest sums (what ``pb200_kv4_compact`` then moves)
  verify    ``pb200_verify_drafts``: drafted tokens against the target's and the draft's logits, by given random numbers: how many are accepted, and the token that follows them

The cache is the one of ``include/prima_b200.h``.  A page holds 64 cells, each a key row and a value row of ``dim`` numbers per layer and head; per layer and head a page is a chunk of
``64 * dim / 2`` bytes of keys, as many of values, and 64 * dim / 32 scales (float16) of each.  A number is ``(n - 8) * scale``, n its 4 bits and the scale that of its block of 32 numbers.
Where bits lie, for cell t (of 64), number d, block b = d / 32 of NB = dim / 32:

  keys      row t of dim / 2 bytes; 32-bit word (d / 8 % 4) * NB + b; of its 8 numbers, number e at bit 4 * (e / 2) + 16 * (e % 2)
  values    row r = t - t % 8 + t % 8 / 2 + 4 * (t % 2); 16-bit word (g ^ (4 * (r / 2 % 2))) * NB + b with g = d / 4 % 8; number d % 4 at bit 4 * (d % 4)
  scales    entry (t / 2 * NB + b) * 2 + t % 2

Verification.  With p and q the target's and the draft's softmax of logits times the sequence's 1 / temperature (infinite: all of it on the largest logit, of several the lowest index; without
draft logits q is all on the drafted token), drafted token x is accepted where u q(x) < p(x), u its given number.  Behind the accepted ones, up to the first that is not, comes a token drawn by
another given number v: from max(p - q, 0) at the place of the rejection (from p, if that is 0 everywhere), from p behind the last one.  It is the lowest i with w_0 + .. + w_i > v * (sum of w).
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
        # eight answers to one question of a thousand tokens, sampled side by side, a layer of an 8B model: the smallest call, one per layer and token
        {"name": "shared_token_8", "kind": "shared", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "groups": "8", "prefix": "1000", "q": "1*8", "kv": "1..120"},
        # 128 requests behind one system prompt of 16 000 tokens and a bit
        {"name": "shared_batch_128", "kind": "shared", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "groups": "128", "prefix": "16009", "q": "1*128", "kv": "5..900"},
        # three tenants, five drafted tokens a request, in 32 bits
        {"name": "shared_groups_f32", "kind": "shared", "type": "f32", "heads": 16, "kv_heads": 4, "dim": 128, "groups": "13,7,4", "prefix": "3001,640,2047", "q": "5*24", "kv": "5..400"},
        # prompts of four requests behind a common document, and one that decodes beside them, heads of 64
        {"name": "shared_prompts_f16", "kind": "shared", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 64, "groups": "5", "prefix": "6000", "q": "700,33,257,512,1", "kv": "700,133,257,512,77"},
        # one generated token of one request: its weights are added up beside it
        {"name": "weigh_token_1000", "kind": "weigh", "type": "f32", "heads": 32, "kv_heads": 8, "dim": 128, "q": "1", "kv": "1001", "window": 0, "first": 0, "decay": 1.0},
        # 32 requests that decode together, older weights fading
        {"name": "weigh_batch_32", "kind": "weigh", "type": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "1*32", "kv": "17..8192", "window": 0, "first": 0, "decay": 0.98},
        # the last 64 queries of two long prompts decide what stays, heads of 64
        {"name": "weigh_prompt_64", "kind": "weigh", "type": "f16", "heads": 16, "kv_heads": 4, "dim": 64, "q": "64,64", "kv": "16384,9001", "window": 0, "first": 0, "decay": 0.0},
        # one request gives up half of a thousand cells
        {"name": "select_1000", "kind": "select", "kv": "1000", "keep": 0.5, "first": 4, "last": 64},
        # a batch of long contexts comes back to a quarter
        {"name": "select_24", "kind": "select", "kv": "300..131072", "seqs": 24, "keep": 0.25, "first": 4, "last": 256},
        # three drafted tokens of one request, by a draft model
        {"name": "verify_1", "kind": "verify", "type": "f32", "vocab": 32000, "drafts": "3", "draft": True, "temp": 0.8},
        # 64 requests of a large vocabulary, ragged drafts
        {"name": "verify_64", "kind": "verify", "type": "f32", "vocab": 128256, "drafts": "4,5,3,0,4,8,1,4", "seqs": 64, "draft": True, "temp": 1.0},
        # drafts from the prompt's own text (no draft model), 16-bit logits of an odd vocabulary, some requests greedy
        {"name": "verify_24_lookup", "kind": "verify", "type": "bf16", "vocab": 151937, "drafts": "2,7,4", "seqs": 24, "draft": False, "temp": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "weigh", "weigh", "select", "verify", "verify"])
    dim, kv_heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8])
    if kind == "shared":
        group = rng.choice([1, 2, 3, 4, 7, 8])
        groups = [_log_int(rng, 1, 40) for _ in range(rng.choice([1, 1, 1, 2, 5]))]
        n = sum(groups)
        if n <= 12 and rng.random() < 0.4:
            q = [rng.choice([1, 5, _log_int(rng, 2, 300)]) for _ in range(n)]
            kv = [a + rng.choice([0, 0, _log_int(rng, 1, 200)]) for a in q]
        else:
            q = [rng.choice([1, 1, 1, 4, 9])] * n
            kv = [a + _log_int(rng, 1, 800) - 1 for a in q]
        most = max(64, min(16000, 60000000 // (sum(q) * group * kv_heads)))
        prefix = [rng.choice([_log_int(rng, 1, most), _log_int(rng, 64, most), 64 * rng.randrange(1, 1 + most // 64)]) for _ in groups]
        return {"kind": "shared", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "groups": ",".join(map(str, groups)),
                "prefix": ",".join(map(str, prefix)), "q": ",".join(map(str, q)), "kv": ",".join(map(str, kv))}
    if kind == "weigh":
        group, n = rng.choice([1, 2, 3, 4, 8]), _log_int(rng, 1, 32)
        q = [rng.choice([1, 1, 1, 4])] * n
        most = _log_int(rng, 8, min(16000, max(16, 250000 * 8 // (n * kv_heads * group))))
        if rng.random() < 0.4:
            q = [_log_int(rng, 2, 400) for _ in range(rng.choice([1, 2, 3]))]
            most = _log_int(rng, 16, max(64, min(16000, 20000000 // (sum(q) * kv_heads * group))))
        kv = [max(a, rng.randrange(1, most + 1)) for a in q]
        return {"kind": "weigh", "type": rng.choice(["f32", "f16", "bf16"]), "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "q": ",".join(map(str, q)), "kv": ",".join(map(str, kv)),
                "window": rng.choice([0, 0, 0, _log_int(rng, 1, 2048)]), "first": rng.choice([0, 4, 65]), "decay": rng.choice([0.0, 1.0, 0.9])}
    if kind == "select":
        n, most = _log_int(rng, 1, 24), _log_int(rng, 2, 100000)
        return {"kind": "select", "kv": "%d..%d" % (max(1, most // rng.choice([1, 3, 40])), most), "seqs": n, "keep": rng.choice([0.02, 0.25, 0.5, 0.9, 1.0]), "first": rng.choice([0, 1, 4, 100]),
                "last": rng.choice([0, 1, 32, 300])}
    n = _log_int(rng, 1, 40)
    return {"kind": "verify", "type": rng.choice(["f32", "f16", "bf16"]), "vocab": _log_int(rng, 500, 160000), "drafts": ",".join(str(rng.choice([0, 1, 2, 3, 4, 5, 7])) for _ in range(n)), "seqs": n,
            "draft": rng.random() < 0.7, "temp": rng.choice([0.0, 0.7, 1.0, 1.3])}


def _numbers(text, n=None):
    """"3,5", "1*4" (four ones) or "3..50" (n numbers between, spread like the multiples of the golden ratio; the last one is the largest); repeated up to n"""
    if ".." in text:
        lo, hi = map(int, text.split(".."))
        lo = min(lo, hi)
        return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) for i in range(n - 1)] + [hi]
    if "*" in text:
        v, k = map(int, text.split("*"))
        return [v] * k
    out = [int(v) for v in text.split(",")]
    return out if n is None else [out[i % len(out)] for i in range(n)]


def _lengths(case):
    q = _numbers(case["q"])
    return q, _numbers(case["kv"], len(q))


def _budgets(case):
    kv = _numbers(case["kv"], case.get("seqs", 1))
    return kv, [max(1, int(round(n * case["keep"]))) for n in kv]


# ---------------------------------------------------------------------------------------------------------------- the cache's format, in elementary operations
def _quantize(x):
    """float32 [..., dim] -> (4 bits each as uint8 [..., dim], scales float16 [..., dim / 32])"""
    b = x.clamp(-21760.0, 21760.0).reshape(*x.shape[:-1], -1, 32)
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


def _unpack_v(raw):
    w = _turn(raw.reshape(*raw.shape[:-2], 8, 8, 8, -1))
    w = w.reshape(*raw.shape[:-2], 8, 2, 4, 8, w.shape[-1]).transpose(-3, -4).reshape(*raw.shape[:-1], 8, -1)
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
    g.manual_seed(0x5EED5 + 6151 * int(seed))
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


def _ints(values):
    return torch.from_numpy(np.asarray(values, dtype=np.int32)).to(DEV)


def _workspace():
    """bytes of the attention's workspace, which a program allocates once, zeroed"""
    return 64 << 20


class _State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    g = _gen(seed)
    S = _State(case=case, kind=case["kind"])
    if case["kind"] in ("shared", "weigh"):
        dim, hk = case["dim"], case["kv_heads"]
        q, kv = _lengths(case)
        prefix = _numbers(case["prefix"]) if case["kind"] == "shared" else []
        table, pool = _tables(g, prefix + kv, 3)
        pages = torch.empty(pool, 1, hk, _chunk(dim), dtype=torch.uint8, device=DEV)
        _fill(g, pages, dim)
        n, tokens = len(prefix), sum(q)
        S.update(n_seq=len(q), max_q=max(q), tokens=tokens, pages=pages, table=table[n:, :max(1, -(-max(kv) // CELLS))].contiguous(), kv_len=_ints(kv),
                 q_start=_ints(np.concatenate(([0], np.cumsum(q)))), q=_randn(g, tokens, case["heads"], dim).to(TYPES[case["type"]]),
                 place=torch.from_numpy(np.concatenate([np.arange(k) + i * max(q) for i, k in enumerate(q)])).to(DEV))
        S["out"] = torch.zeros_like(S["q"])
        S["lse"] = torch.zeros(tokens, case["heads"], device=DEV)
        S["ws"] = torch.zeros(_workspace() + (4 * tokens * case["heads"] * (dim + 2) if n else 0), dtype=torch.uint8, device=DEV)
        if n:
            groups = _numbers(case["groups"])
            S.update(prefix_table=table[:n, :max(1, -(-max(prefix) // CELLS))].contiguous(), prefix_len=_ints(prefix), group_start=_ints(np.concatenate(([0], np.cumsum(groups)))),
                     prefix=prefix, rows=np.concatenate(([0], np.cumsum(q)))[np.concatenate(([0], np.cumsum(groups)))].tolist())
        else:
            # what earlier tokens left: a few cells have most of it
            S["old"] = torch.rand(len(q), max(kv), generator=g, device=DEV).pow(8) * 40.0
            S["sums"] = torch.zeros_like(S["old"])
    elif case["kind"] == "select":
        kv, budget = _budgets(case)
        weight = torch.rand(len(kv), max(kv), generator=g, device=DEV).pow(8) * 40.0
        weight = torch.where(torch.rand(weight.shape, generator=g, device=DEV) < 0.1, 0.0, weight)            # cells that a window hides have none
        S.update(n_seq=len(kv), sums=weight, kv_len=_ints(kv), budget=_ints(budget), max_len=max(kv), most=max(budget),
                 index=torch.zeros(len(kv), max(budget), dtype=torch.int32, device=DEV), count=torch.zeros(len(kv), dtype=torch.int32, device=DEV),
                 kept=torch.zeros(len(kv), max(budget), device=DEV))
    else:
        drafts = _numbers(case["drafts"], case.get("seqs", 1))
        n, total, vocab, t = len(drafts), sum(drafts), case["vocab"], TYPES[case["type"]]
        start = np.concatenate(([0], np.cumsum(drafts)))
        S.update(n_seq=n, drafts=total, start=_ints(start), most=max(drafts) + 1)
        S["seq"] = torch.from_numpy(np.repeat(np.arange(n), drafts)).to(DEV)                                # of each draft
        S["target"] = (_randn(g, total + n, vocab) * 2.5).to(t)
        # a draft model that agrees for the most part; without one the drafts are likely tokens
        row = torch.arange(total, device=DEV) + S["seq"]
        logits = torch.empty(total, vocab, dtype=t, device=DEV)
        tokens = torch.empty(total, dtype=torch.int32, device=DEV)
        S["inv_temp"] = torch.full((n,), 1.0 / case["temp"] if case["temp"] else 1.0, device=DEV)
        if not case["temp"]:
            S["inv_temp"][::2] = math.inf
        for i in range(total):
            x = S["target"][row[i]].float() + 0.7 * _randn(g, vocab)
            logits[i] = x.to(t)
            noise = -torch.log(-torch.log(torch.rand(vocab, generator=g, device=DEV, dtype=torch.float64).clamp(1e-300, 1.0 - 1e-16)))
            temp = S["inv_temp"][S["seq"][i]].double()
            tokens[i] = torch.where(torch.isinf(temp), logits[i].double(), logits[i].double() * temp + noise).argmax().to(torch.int32)
        S.update(tokens=tokens, draft=logits if case["draft"] else None, u=torch.rand(total, generator=g, device=DEV), v=torch.rand(n, generator=g, device=DEV),
                 kv_len=_ints(np.arange(n) * 37 % 4096 + 50), kv_out=torch.zeros(n, dtype=torch.int32, device=DEV), accepted=torch.zeros(n, dtype=torch.int32, device=DEV),
                 out=torch.full((n, S["most"]), -1, dtype=torch.int32, device=DEV), ws=torch.zeros((1 << 20) + 4096 * (total + n), dtype=torch.uint8, device=DEV))
    return S


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _rows_of(S):
    """queries float32 [n_seq, kv_heads, max_q * group, dim]"""
    c = S.case
    hk, grp, dim = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    q = torch.zeros(S.n_seq * S.max_q, c["heads"], dim, device=DEV)
    q[S.place] = S.q.float()
    return q.reshape(S.n_seq, S.max_q, hk, grp, dim).permute(0, 2, 1, 3, 4).reshape(S.n_seq, hk, S.max_q * grp, dim)


def _tokens_of(S, x):
    """[n_seq, kv_heads, max_q * group, k] -> [tokens, heads, k]"""
    c = S.case
    hk, grp = c["kv_heads"], c["heads"] // c["kv_heads"]
    return x.reshape(S.n_seq, hk, S.max_q, grp, -1).permute(0, 2, 1, 3, 4).reshape(S.n_seq * S.max_q, c["heads"], -1)[S.place]


def _keys_values(S, table):
    c = S.case
    raw = S.pages[table.clamp(min=0).long(), 0]                                                           # n, pages, heads, bytes
    return (x.transpose(1, 2).reshape(table.shape[0], c["kv_heads"], -1, c["dim"]) for x in _page_values(raw, c["dim"]))


def _own_cells(S):
    """scores (-inf where not seen) [n_seq, kv_heads, max_q * group, cells] of the sequences' own cells, and the values"""
    c = S.case
    k, v = _keys_values(S, S.table)
    s = torch.matmul(_rows_of(S), k.transpose(-1, -2)) * (1.0 / math.sqrt(c["dim"]))
    n_q = (S.q_start[1:] - S.q_start[:-1])[:, None, None]
    p = S.kv_len[:, None, None] - n_q + torch.arange(S.max_q, device=DEV)[None, :, None]
    i = torch.arange(k.shape[2], device=DEV)[None, None, :]
    see = (i <= p) & (torch.arange(S.max_q, device=DEV)[None, :, None] < n_q)
    if c.get("window"):
        see = see & ((p - i < c["window"]) | (i < c["first"]))
    see = see[:, None, :, None, :].expand(-1, 1, -1, c["heads"] // c["kv_heads"], -1).reshape(S.n_seq, 1, -1, k.shape[2])
    return torch.where(see, s, -math.inf), v


def _weights(s):
    """largest score (0 where nothing is seen), weights, and their sum"""
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    w = torch.exp(s - m)
    return m, w, w.sum(-1, keepdim=True)


def _plain_shared(S):
    c = S.case
    hk, grp, dim = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    s, v = _own_cells(S)
    m, w, total = (_tokens_of(S, x) for x in (lambda m, w, t: (m, torch.matmul(w, v), t))(*_weights(s)))
    out = torch.empty(S.tokens, c["heads"], dim, device=DEV)
    lse = torch.empty(S.tokens, c["heads"], device=DEV)
    for i, length in enumerate(S.prefix):
        a, b = S.rows[i], S.rows[i + 1]
        k, v = (x[0, :, :length] for x in _keys_values(S, S.prefix_table[i:i + 1]))
        q = S.q[a:b].float().reshape(b - a, hk, grp, dim).transpose(0, 1).reshape(hk, -1, dim)
        pm, pw, pt = _weights(torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim)))
        pm, pw, pt = (x.reshape(hk, b - a, grp, -1).transpose(0, 1).reshape(b - a, c["heads"], -1) for x in (pm, torch.matmul(pw, v), pt))
        top = torch.where(total[a:b] == 0, pm, torch.maximum(m[a:b], pm))
        f, pf = torch.exp(m[a:b] - top) * (total[a:b] > 0), torch.exp(pm - top)
        both = total[a:b] * f + pt * pf
        out[a:b] = (w[a:b] * f + pw * pf) / both
        lse[a:b] = (top + torch.log(both)).squeeze(-1)
    return [out.to(S.q.dtype), lse]


def _plain_weigh(S):
    c = S.case
    s, v = _own_cells(S)
    m, w, total = _weights(s)
    some = torch.where(total == 0, 1.0, total)
    lse = torch.where(total == 0, -math.inf, m + torch.log(some))
    sums = (w / some).sum((1, 2))[:, :S.old.shape[1]] + c["decay"] * S.old
    sums = torch.where(torch.arange(S.old.shape[1], device=DEV) < S.kv_len[:, None], sums, 0.0)
    return [_tokens_of(S, torch.matmul(w, v) / some).to(S.q.dtype), _tokens_of(S, lse).squeeze(-1), sums]


def _plain_select(S):
    c = S.case
    n, width = S.sums.shape
    j = torch.arange(width, device=DEV)[None]
    count = torch.minimum(S.kv_len, S.budget)[:, None]
    last = torch.clamp(count, max=c["last"])
    first = torch.minimum(count - last, torch.full_like(count, c["first"]))
    length = S.kv_len[:, None]
    # the cells of a sequence in the order in which they stay: the first and last ones, then by their sums, of equal ones the lowest
    always = (j < first) | ((j >= length - last) & (j < length))
    key = torch.where(always, math.inf, torch.where(j < length, S.sums, -math.inf))
    rank = torch.empty_like(key, dtype=torch.long)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank.scatter_(1, order, j.expand(n, -1))
    keep = rank < count
    at = torch.cumsum(keep, 1) - 1
    index, kept = torch.zeros_like(S.index), torch.zeros_like(S.kept)
    row, col = keep.nonzero(as_tuple=True)
    index[row, at[row, col]] = col.to(torch.int32)
    kept[row, at[row, col]] = S.sums[row, col]
    return [index, count.squeeze(1).to(torch.int32), kept]


def _softmax64(logits, inv_temp):
    """float64; all of it on the first of the largest where 1 / temperature is infinite"""
    x = logits.double()
    d = x - x.amax(-1, keepdim=True)
    t = inv_temp.double()[:, None]
    e = torch.exp(torch.where(torch.isinf(t), 0.0, t) * d)
    top = torch.zeros_like(e).scatter_(1, x.argmax(-1, keepdim=True), 1.0)
    e = torch.where(torch.isinf(t), top, e)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(S):
    c = S.case
    n, vocab = S.n_seq, c["vocab"]
    row = torch.arange(S.drafts, device=DEV) + S.seq
    token = S.tokens.long()[:, None]
    n_draft = S.start[1:] - S.start[:-1]
    ok = torch.zeros(n, S.most, dtype=torch.bool, device=DEV)
    col = torch.arange(S.drafts, device=DEV) - S.start[:-1].long()[S.seq]
    if S.drafts:
        p = _softmax64(S.target[row], S.inv_temp[S.seq])
        q = _softmax64(S.draft, S.inv_temp[S.seq]) if S.draft is not None else torch.zeros_like(p).scatter_(1, token, 1.0)
        ok[S.seq, col] = S.u.double() * q.gather(1, token).squeeze(1) < p.gather(1, token).squeeze(1)
    accepted = torch.cumprod(ok.int(), 1).sum(1)
    # the rows that the next tokens are drawn from
    at = S.start[:-1] + accepted
    w = _softmax64(S.target[at + torch.arange(n, device=DEV)], S.inv_temp)
    if S.drafts:
        rest = torch.clamp(w - q[at.clamp(max=S.drafts - 1)], min=0.0)
        w = torch.where(((accepted < n_draft) & (rest.sum(-1) > 0))[:, None], rest, w)
    cum = torch.cumsum(w, -1)
    x = S.v.double()[:, None] * cum[:, -1:]
    last = vocab - 1 - (w.flip(-1) > 0).int().argmax(-1)
    drawn = torch.where(cum[:, -1:] > x, cum > x, False).int().argmax(-1)
    drawn = torch.where(cum[:, -1] > x[:, 0], drawn, last)
    out = torch.full((n, S.most), -1, dtype=torch.int32, device=DEV)
    taken = col < accepted[S.seq]
    out[S.seq[taken], col[taken]] = S.tokens[taken]
    out[torch.arange(n, device=DEV), accepted] = drawn.to(torch.int32)
    return [accepted.to(torch.int32), out, (S.kv_len - n_draft + accepted).to(torch.int32)]


# ---------------------------------------------------------------------------------------------------------------- the framework's operators
def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _own(S):
    import pkgload
    pkg = pkgload.load()
    lib = pkg.Lib.get()
    c, stream = S.case, C.c_void_p(torch.cuda.current_stream().cuda_stream)
    if S.kind in ("shared", "weigh"):
        h, dim, code = c["heads"], c["dim"], CODES[c["type"]]
        cache = pkg.Kv4Cache(S.pages.data_ptr(), S.pages.shape[0], S.pages.shape[1], S.pages.shape[2], dim)
        scale = 1.0 / math.sqrt(dim)
        if S.kind == "shared":
            lib.check(lib.c.pb200_kv4_attn_shared(C.byref(cache), 0, code, _p(S.q), h * dim, _p(S.out), h * dim, h, S.n_seq, _p(S.q_start), _p(S.kv_len), _p(S.table), S.table.shape[1],
                                                  S.prefix_len.shape[0], _p(S.group_start), _p(S.prefix_len), _p(S.prefix_table), S.prefix_table.shape[1], S.tokens, S.max_q, scale, _p(S.lse), h,
                                                  _p(S.ws), S.ws.numel(), stream), "kv4_attn_shared")
            return [S.out, S.lse]
        lib.check(lib.c.pb200_kv4_attn_lse(C.byref(cache), 0, code, _p(S.q), h * dim, _p(S.out), h * dim, h, S.n_seq, _p(S.q_start), _p(S.kv_len), _p(S.table), S.table.shape[1], S.tokens,
                                           S.max_q, scale, c["window"], c["first"], _p(S.lse), h, _p(S.ws), S.ws.numel(), stream), "kv4_attn_lse")
        lib.check(lib.c.pb200_kv4_weigh(C.byref(cache), 0, code, _p(S.q), h * dim, h, S.n_seq, _p(S.q_start), _p(S.kv_len), _p(S.table), S.table.shape[1], S.tokens, S.max_q, scale, c["window"],
                                        c["first"], _p(S.lse), h, c["decay"], _p(S.old), S.old.shape[1], _p(S.sums), S.sums.shape[1], stream), "kv4_weigh")
        return [S.out, S.lse, S.sums]
    if S.kind == "select":
        lib.check(lib.c.pb200_kv4_select(S.n_seq, _p(S.sums), S.sums.shape[1], _p(S.kv_len), S.max_len, _p(S.budget), c["first"], c["last"], _p(S.index), S.index.shape[1], _p(S.count),
                                         _p(S.kept), S.kept.shape[1], stream), "kv4_select")
        return [S.index, S.count, S.kept]
    lib.check(lib.c.pb200_verify_drafts(CODES[c["type"]], _p(S.target), c["vocab"], _p(S.draft), c["vocab"], c["vocab"], S.n_seq, _p(S.start), S.drafts, _p(S.tokens), _p(S.inv_temp), _p(S.u), _p(S.v),
                                        _p(S.accepted), _p(S.out), S.most, _p(S.kv_len), _p(S.kv_out), _p(S.ws), S.ws.numel(), stream), "verify_drafts")
    return [S.accepted, S.out, S.kv_out]


def run(state):
    if own:
        return _own(state)
    return {"shared": _plain_shared, "weigh": _plain_weigh, "select": _plain_select, "verify": _plain_verify}[state.kind](state)


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def _seen(p, window, first):
    """cells that the query at position p sees"""
    if p < 0:
        return 0
    if window == 0 or p + 1 <= window:
        return p + 1
    return window + min(first, p + 1 - window)


def work(case):
    size = 4 if case.get("type") == "f32" else 2
    if case["kind"] in ("shared", "weigh"):
        dim, hk, window, first = case["dim"], case["kv_heads"], case.get("window", 0), case.get("first", 0)
        row = dim // 2 + dim // 16
        q, kv = _lengths(case)
        cells = pairs = 0
        for n, length in zip(q, kv):
            p0 = length - n
            pairs += sum(_seen(p0 + i, window, first) for i in range(n))
            lo = max(0, p0 - window + 1) if window else 0
            cells += length - lo + min(lo, first)
        if case["kind"] == "shared":
            at = 0
            for n, length in zip(_numbers(case["groups"]), _numbers(case["prefix"])):
                cells += length
                pairs += length * sum(q[at:at + n])
                at += n
        sums = 8 * sum(kv) if case["kind"] == "weigh" else 0
        return {"bytes": 2 * sum(q) * case["heads"] * dim * size + 4 * sum(q) * case["heads"] + cells * hk * 2 * row + sums, "flops": 4 * pairs * case["heads"] * dim}
    if case["kind"] == "select":
        kv, budget = _budgets(case)
        return {"bytes": 4 * sum(kv) + 8 * sum(min(a, b) for a, b in zip(kv, budget)), "flops": 0}
    drafts = _numbers(case["drafts"], case.get("seqs", 1))
    # rows of the drafts, and one more where all are accepted, which a pass may have to read
    rows = sum(drafts) * (2 if case["draft"] else 1) + len(drafts)
    return {"bytes": rows * case["vocab"] * size, "flops": 4 * rows * case["vocab"]}


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


def exact(case, seed):
    if case["kind"] in ("select", "verify"):
        return None                      # whole numbers, and numbers that move; both sides draw tokens in 64 bits
    S = prepare(case, seed)
    dim, hk = case["dim"], case["kv_heads"]
    q_len, kv_len = _lengths(case)
    grp, shared = case["heads"] // hk, case["kind"] == "shared"
    kb, ksh, vb, vsh, sc = _place(dim)

    def read(ids, j, length):
        raw, k, v = S.pages[ids.long(), 0, j], [], []
        for i in range(0, raw.shape[0], 256):
            k.append(_value(raw[i:i + 256], kb, ksh, sc))
            v.append(_value(raw[i:i + 256], vb, vsh, sc + CELLS * dim // 16))
        return [torch.cat(z).reshape(-1, dim)[:length] if z else torch.zeros(0, dim, dtype=torch.float64, device=DEV) for z in (k, v)]

    group_of = np.repeat(np.arange(len(S.prefix)), _numbers(case["groups"])) if shared else None
    out = torch.zeros(S.tokens, case["heads"], dim, dtype=torch.float64, device=DEV)
    lse = torch.zeros(S.tokens, case["heads"], dtype=torch.float64, device=DEV)
    sums = None if shared else torch.zeros(S.old.shape, dtype=torch.float64, device=DEV)
    for j in range(hk):
        at, held = 0, None
        for s, (n, length) in enumerate(zip(q_len, kv_len)):
            k, v = read(S.table[s, :-(-length // CELLS)], j, length)
            front = 0
            if shared:
                if held is None or held[0] != group_of[s]:
                    front = S.prefix[group_of[s]]
                    held = (group_of[s], *read(S.prefix_table[group_of[s], :-(-front // CELLS)], j, front))
                front = S.prefix[group_of[s]]
                k, v = torch.cat((held[1], k)), torch.cat((held[2], v))
            cell = torch.arange(front + length, device=DEV) - front
            for i in range(0, n, 512):
                m = min(512, n - i)
                p = length - n + i + torch.arange(m, device=DEV)[:, None]
                hide = cell > p
                if case.get("window"):
                    hide |= (cell <= p - case["window"]) & (cell >= case["first"])
                z = torch.einsum("thd,cd->htc", S.q[at + i:at + i + m, j * grp:(j + 1) * grp].double(), k) / math.sqrt(dim)
                z = z.masked_fill(hide & (cell >= 0), -math.inf)
                w = torch.softmax(z, -1).nan_to_num(0.0)
                out[at + i:at + i + m, j * grp:(j + 1) * grp] = torch.einsum("htc,cd->thd", w, v)
                lse[at + i:at + i + m, j * grp:(j + 1) * grp] = torch.logsumexp(z, -1).T
                if not shared:
                    sums[s, :length] += w.sum((0, 1))
            if not shared and j == 0:
                sums[s, :length] += float(np.float32(case["decay"])) * S.old[s, :length].double()
            at += n
    return [out, lse] if shared else [out, lse, sums]
