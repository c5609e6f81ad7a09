"""The cache of 4-bit keys and values (include/prima_b200.h, csrc/kv4.cuh) in 64 bits: where its bits lie, number by number, and what its operators compute."""
import numpy as np

CELLS = 64
CODE = {"f32": 0, "f16": 1, "bf16": 30}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # of a rounding, relative to the value


def chunk_bytes(dim):
    return 2 * (CELLS * dim // 2 + CELLS * dim // 16)


def places(dim):
    """(byte, shift) of number d of cell t for keys and values, the byte of its scale for both: [64, dim] each"""
    nb, rows, sc = dim // 32, CELLS * dim // 2, CELLS * dim // 16
    kb, ks, vb, vs, s = (np.zeros((CELLS, dim), np.int64) for _ in range(5))
    for t in range(CELLS):
        r = t // 8 * 8 + t % 8 // 2 + 4 * (t % 2)
        for d in range(dim):
            e = d % 8
            bit = 32 * ((d // 8 % 4) * nb + d // 32) + 4 * (e // 2) + 16 * (e % 2)
            kb[t, d], ks[t, d] = t * dim // 2 + bit // 8, bit % 8
            bit = 16 * (((d // 4 % 8) ^ (4 * (r // 2 % 2))) * nb + d // 32) + 4 * (d % 4)
            vb[t, d], vs[t, d] = rows + r * dim // 2 + bit // 8, bit % 8
            s[t, d] = 2 * rows + 2 * ((t // 2 * nb + d // 32) * 2 + t % 2)
    return kb, ks, vb, vs, s, s + sc


def round_bits(x, bits):
    man, exp = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.rint(np.ldexp(man, bits)), exp - bits)


def quantize(x):
    """float64 [..., dim] -> (n 0 .. 15, scale by block)"""
    x = np.where(np.isnan(x), 0.0, np.clip(x, -21760.0, 21760.0)).reshape(*x.shape[:-1], -1, 32)
    most = np.take_along_axis(x, np.abs(x).argmax(-1)[..., None], -1)
    scale = round_bits(most / -8.0, 8).astype(np.float16).astype(np.float64)
    q = np.float32(x) / np.where(scale == 0, 1.0, scale).astype(np.float32)        # the quotient in 32 bits, as the format defines it
    n = np.where(scale == 0, 8, np.clip(np.rint(q.astype(np.float32)) + 8, 0, 15)).astype(np.uint8)
    return n.reshape(*n.shape[:-2], -1), scale[..., 0]


def values(n, scale):
    return (n.astype(np.float64) - 8.0) * np.repeat(scale, 32, -1)


def pack(kn, ks, vn, vs):
    """bits [..., 64, dim] and scales [..., 64, dim / 32] -> chunks"""
    dim = kn.shape[-1]
    kb, ksh, vb, vsh, ksc, vsc = places(dim)
    out = np.zeros((*kn.shape[:-2], chunk_bytes(dim)), np.uint8)
    flat, kn, vn = out.reshape(-1, out.shape[-1]), kn.reshape(-1, CELLS, dim), vn.reshape(-1, CELLS, dim)
    ks16, vs16 = (np.ascontiguousarray(s, dtype=np.float16).reshape(-1, CELLS, dim // 32).view(np.uint16) for s in (ks, vs))
    for shift in (0, 4):
        for n, b, sh in ((kn, kb, ksh), (vn, vb, vsh)):
            at = sh == shift
            flat[:, b[at]] |= n[:, at] << shift
    for s16, sc in ((ks16, ksc), (vs16, vsc)):
        at = sc[:, ::32]
        flat[:, at] = s16 & 255
        flat[:, at + 1] = s16 >> 8
    return out


def unpack(raw, dim):
    """chunks -> keys and values [..., 64, dim] in 64 bits"""
    kb, ksh, vb, vsh, ksc, vsc = places(dim)
    flat = raw.reshape(-1, raw.shape[-1])
    out = []
    for b, sh, sc in ((kb, ksh, ksc), (vb, vsh, vsc)):
        s = (flat[:, sc].astype(np.uint16) | flat[:, sc + 1].astype(np.uint16) << 8).view(np.float16).astype(np.float64)
        out.append((((flat[:, b] >> sh) & 15).astype(np.float64) - 8.0) * s)
    return [x.reshape(*raw.shape[:-1], CELLS, dim) for x in out]


def attend(q, pages, table, q_start, kv_len, n_head_kv, dim, scale, window=0, first=0):
    """q float64 [tokens, heads, dim], pages uint8 [pages, heads, bytes] of a layer -> (out, bound of the error of a kernel with 32-bit sums, largest sum of a
    score's magnitudes); rows without a sequence NaN.

    The bound: a score is a sum of dim products, each rounded and added with 2^-23 of the sum of magnitudes at most, twice that for operands of 22 bits; a weight is
    off by its score's error, 2^-22 of the exponential and 2^-23 of its argument, |score| times that; the sums run over steps of 16 cells and 64 parts."""
    out = np.full(q.shape, np.nan)
    bound, reach = np.zeros(q.shape), 0.0
    group = q.shape[1] // n_head_kv
    for s in range(len(kv_len)):
        n = q_start[s + 1] - q_start[s]
        length = max(int(kv_len[s]), 0)
        need = min(-(-length // CELLS), table.shape[1])
        cells = np.arange(need * CELLS)
        ids = table[s, :need]
        ok = np.repeat((ids >= 0) & (ids < len(pages)), CELLS)
        with np.errstate(invalid="ignore", over="ignore"):
            k, v = unpack(pages[np.where((ids >= 0) & (ids < len(pages)), ids, 0)], dim) if need else [np.zeros((0, n_head_kv, CELLS, dim))] * 2
        k, v = (x.transpose(1, 0, 2, 3).reshape(n_head_kv, -1, dim) for x in (k, v))
        for i in range(n):
            p = int(kv_len[s]) - n + i
            see = ok & (cells <= p)
            if window:
                see = see & ((p - cells < window) | (cells < first))
            row = q_start[s] + i
            out[row] = 0.0
            if not see.any():
                continue
            for h in range(n_head_kv):
                kk, vv, qq = k[h][see], v[h][see], q[row, h * group:(h + 1) * group]
                z = qq @ kk.T * scale
                w = np.exp(z - z.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                out[row, h * group:(h + 1) * group] = w @ vv
                mag = (np.abs(qq) @ np.abs(kk).T).max(-1) * abs(scale)
                reach = max(reach, float(mag.max()))
                rel = 2 * (dim + 8) * 2.0 ** -23 * mag + np.abs(z).max(-1) * 2.0 ** -22 + 2.0 ** -20 + (see.sum() / 16 + 64) * 2.0 ** -23
                bound[row, h * group:(h + 1) * group] = (rel * np.abs(vv).max())[:, None]
    return out, bound, reach


def append(x, weight, eps, pos, w, mode, n_dims, mscale=1.0):
    """rows [tokens, heads, dim] normed (weight not None) and rotated by pos * w, in 64 bits"""
    y = np.array(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + float(np.float32(eps))) * weight
    for i in range(n_dims // 2):
        a, b = (2 * i, 2 * i + 1) if mode == 0 else (i, i + n_dims // 2)
        ang = pos.astype(np.float64) * w[i]
        c, s = (np.cos(ang) * mscale)[:, None], (np.sin(ang) * mscale)[:, None]
        y[..., a], y[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    return y
