"""CPU restatement of the sparse-attention operators (test infrastructure only): the tables of a
step, block choice by the indexer's scores, the 4-bit MLA slot, and MLA attention over selected
tokens, in numpy with 64-bit floats and integers, written from the definitions."""
from __future__ import annotations

import numpy as np

PAGE, LATENT, ROPE = 64, 512, 64
FP8_SLOT, KV4_SLOT = 656, 432
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], np.float64)


def bf16_to_f64(u16):
    return (np.asarray(u16, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def _e4m3_table():
    v = np.empty(256, np.float64)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[b] = -x if b & 128 else x
        if (b & 127) == 127:
            v[b] = np.nan
    return v


E4M3 = _e4m3_table()


def e4m3_round(x):
    """Nearest e4m3 of x >= 0 (ties to even, saturated) -> codes."""
    x = np.asarray(x, np.float64)
    pos = E4M3[:127]
    hi = np.clip(np.searchsorted(pos, x), 1, 126)
    lo = hi - 1
    dl, dh = x - pos[lo], pos[hi] - x
    return np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo).astype(np.uint8)


def e2m1_round(x):
    """Nearest e2m1 of x >= 0 (ties to the even code, saturated) -> codes 0..7."""
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x = np.asarray(x, np.float64)[..., None]
    up = np.where(np.arange(7) % 2 == 0, x > mids, x >= mids)  # code c + 1 is even for odd c
    return up.sum(-1).astype(np.uint8)


def kv4_values(slots):
    """[n, >= 432] bytes -> [n, 576] float64."""
    s = np.ascontiguousarray(slots[:, :KV4_SLOT])
    n = s.shape[0]
    v = np.empty((n, LATENT))
    v[:, 0::2], v[:, 1::2] = E2M1[s[:, :256] & 15], E2M1[s[:, :256] >> 4]
    t = np.ascontiguousarray(s[:, 288:292]).view(np.float32).astype(np.float64)
    v *= np.repeat(E4M3[s[:, 256:288]], 16, axis=1) * t
    return np.concatenate([v, bf16_to_f64(np.ascontiguousarray(s[:, 304:432]).view(np.uint16))], 1)


def fp8_values(slots):
    s = np.ascontiguousarray(slots[:, :FP8_SLOT])
    sc = np.ascontiguousarray(s[:, 512:528]).view(np.float32).astype(np.float64)
    v = E4M3[s[:, :512]] * np.repeat(sc, 128, axis=1)
    return np.concatenate([v, bf16_to_f64(np.ascontiguousarray(s[:, 528:656]).view(np.uint16))], 1)


def kv4_pack(latent_u16, rope_u16):
    """bf16 bits [n, 512] and [n, 64] -> [n, 432] bytes (zeros always as code 0)."""
    x = bf16_to_f64(latent_u16).reshape(-1, 32, 16)
    amax = np.abs(x).max(-1)
    top = amax.max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 11, -100).clip(min=-100)
    t = np.ldexp(1.0, e)
    sg = e4m3_round(np.minimum(amax / t[:, None] / 6, 448))
    s = E4M3[sg] * t[:, None]
    a = np.where(s[..., None] > 0, np.abs(x) / np.where(s > 0, s, 1)[..., None], 0)
    code = e2m1_round(a)
    code = np.where((x < 0) & (code > 0), code + 8, code).astype(np.uint8).reshape(-1, 256, 2)
    n = x.shape[0]
    return np.concatenate([code[..., 0] | (code[..., 1] << 4), sg, t.astype(np.float32).reshape(n, 1).view(np.uint8),
                           np.zeros((n, 12), np.uint8),
                           np.ascontiguousarray(rope_u16).view(np.uint8).reshape(n, 128)], 1)


def block_slots(idx, table, length):
    """Slots of the visible tokens of the listed blocks of one row."""
    out = []
    for b in idx:
        if b < 0:
            continue
        for j in range(PAGE):
            if b * PAGE + j < length:
                out.append(int(table[b]) * PAGE + j)
    return np.array(out, np.int64)


def attend(q, k, sm_scale, eps_k):
    """One row: q [H, 576], k [n, 576] float64 -> (out [H, 512], lse [H], out bound, lse bound).

    The bounds are for products whose k operands carry relative errors of at most eps_k each for a
    factor common to a 128-element group and for a rounding of every element (the rope counting as
    one group): a group's score moves by eps_k of itself at most, and the independent roundings
    (rms eps_k / sqrt(3)) add up in quadrature, six of their standard deviations allowed; 2^-20 of
    sum |q k| stands for the 32-bit accumulation.  d, the largest score error, moves every weight
    by a factor within exp(+-2 d); values carry 2 eps_k, weights 2^-11 (f16) and the result half a
    bf16 step."""
    h = q.shape[0]
    if k.shape[0] == 0:
        return np.zeros((h, LATENT)), np.full(h, -np.inf), np.zeros((h, LATENT)), np.zeros(h)
    s = sm_scale * (q @ k.T)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    z = p.sum(-1, keepdims=True)
    w = p / z
    out = w @ k[:, :LATENT]
    groups = sum(np.abs(q[:, a:b] @ k[:, a:b].T) for a, b in ((0, 128), (128, 256), (256, 384), (384, 512), (512, 576)))
    d = sm_scale * (eps_k * groups + 6 * eps_k / 3 ** 0.5 * np.sqrt((q ** 2) @ (k ** 2).T)
                    + 2.0 ** -20 * (np.abs(q) @ np.abs(k).T))
    d = d.max(-1, keepdims=True)
    spread = w @ np.abs(k[:, :LATENT])
    tol = (2 * d + 2 * eps_k + 2.0 ** -11) * 1.05 * spread + 2.0 ** -8 * 1.01 * np.abs(out) + 1e-30
    return out, (m + np.log(z))[:, 0], tol, d[:, 0] + 2.0 ** -20 * (1 + np.abs(m[:, 0] + np.log(z[:, 0])))


def select_blocks(score, visible_bits, length, n, n_sink, n_local):
    """One row: score [width] with its mask bits -> the n chosen blocks, ascending, -1 pads."""
    nb = -(-length // PAGE)
    best = []
    for b in range(nb):
        t = slice(b * PAGE, min((b + 1) * PAGE, length))
        best.append(np.where(visible_bits[t], score[t], 0.0).max())
    forced = [b < n_sink or b >= nb - n_local for b in range(nb)]
    order = sorted(range(nb), key=lambda b: (not forced[b], 0 if forced[b] else -best[b], b))[:n]
    return np.array(sorted(order) + [-1] * (n - len(order)), np.int32)


def step_tables(req_pages, req_idx, seq, new, free_pages, head, n_rows, width):
    """-> dict of the op's outputs and the updated req_pages."""
    rp = np.array(req_pages, np.int32)
    bt = np.full((n_rows, width // PAGE), -1, np.int32)
    pt = np.full((n_rows, width), -1, np.int32)
    lens, pos, loc = np.zeros(n_rows, np.int32), np.zeros(n_rows, np.int32), np.full(n_rows, -1, np.int64)
    r = 0
    for i, row in enumerate(req_idx):
        have, total = -(-int(seq[i]) // PAGE), -(-int(seq[i] + new[i]) // PAGE)
        for p in range(have, total):
            rp[row, p] = free_pages[head] if head < len(free_pages) else -1
            head += 1
        for j in range(int(new[i])):
            np_ = min(total, width // PAGE)
            bt[r, :np_] = rp[row, :np_]
            t = np.arange(min(int(seq[i] + new[i]), width))
            page = rp[row, t // PAGE]
            pt[r, :len(t)] = np.where(page >= 0, page * PAGE + t % PAGE, -1)
            pos[r] = seq[i] + j
            lens[r] = min(pos[r] + 1, width)
            pg = rp[row, pos[r] // PAGE]
            loc[r] = int(pg) * PAGE + pos[r] % PAGE if pg >= 0 else -1
            r += 1
    return dict(block_table=bt, page_table_size_1=pt, lengths=lens, positions=pos, token_loc=loc.astype(np.int32),
                loc=loc, free_head=np.array([head], np.int32), req_pages=rp)
