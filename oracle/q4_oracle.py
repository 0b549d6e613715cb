"""CPU restatement of the 4-bit cache, its decode attention and token eviction (test infrastructure).

Rows are encoded in IEEE fp32 as the format defines them; attention is in 64 bits over the values that the rows stand
for; eviction sorts. Written in numpy, head by head, from the definitions in include/emm_kv.h.
"""
from __future__ import annotations

import numpy as np

GROUP = 32


def row_bytes(D: int) -> int:
    return -(-(D // 2 + 4 * (D // GROUP)) // 16) * 16


def encode_rows(x: np.ndarray) -> np.ndarray:
    """fp32 values [N, D] (exactly the 16-bit inputs) -> bytes [N, row_bytes(D)]."""
    x = np.asarray(x, dtype=np.float32)
    N, D = x.shape
    G = D // GROUP
    g = x.reshape(N, G, GROUP)
    nan = np.isnan(g).any(-1)
    g = np.clip(np.where(nan[..., None], np.float32(0), g), np.float32(-65504), np.float32(65504))
    lo, hi = g.min(-1), g.max(-1)
    s = ((hi - lo) / np.float32(15)).astype(np.float16)
    o = (lo + np.float32(8) * s.astype(np.float32)).astype(np.float16)
    sf, of = s.astype(np.float32)[..., None], o.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((g - of) / sf)
    c = np.clip(np.where(sf == 0, np.float32(0), q) + 8, 0, 15).astype(np.uint8)
    c[nan] = 8
    bits_s, bits_o = s.view(np.uint16).copy(), o.view(np.uint16).copy()
    bits_s[nan], bits_o[nan] = 0, 0x7FFF
    out = np.zeros((N, row_bytes(D)), dtype=np.uint8)
    for d in range(D):
        r, u, i = d // GROUP, d % GROUP // 4, d % 4
        out[:, 2 * (u * G + r) + i // 2] |= c[:, r, d % GROUP] << (4 * (i % 2))
    out[:, D // 2: D // 2 + 2 * G] = bits_s.view(np.uint8)
    out[:, D // 2 + 2 * G: D // 2 + 4 * G] = bits_o.view(np.uint8)
    return out


def decode_parts(rows: np.ndarray, D: int):
    """Bytes [..., row_bytes(D)] -> (offset, scale * (code - 8)) per channel, in 64 bits."""
    rows = np.ascontiguousarray(rows)
    G = D // GROUP
    d = np.arange(D)
    r, u, i = d // GROUP, d % GROUP // 4, d % 4
    byte = rows[..., 2 * (u * G + r) + i // 2]
    code = np.where(i % 2 == 1, byte >> 4, byte & 15).astype(np.float64)
    s = np.ascontiguousarray(rows[..., D // 2: D // 2 + 2 * G]).view(np.float16).astype(np.float64)
    o = np.ascontiguousarray(rows[..., D // 2 + 2 * G: D // 2 + 4 * G]).view(np.float16).astype(np.float64)
    return o[..., r], s[..., r] * (code - 8.0)


def code_part(rows: np.ndarray, D: int) -> np.ndarray:
    """scale * code per channel, in 64 bits."""
    _, v = decode_parts(rows, D)
    G = D // GROUP
    s = np.ascontiguousarray(np.ascontiguousarray(rows)[..., D // 2: D // 2 + 2 * G]).view(np.float16).astype(np.float64)
    return v + 8.0 * s[..., np.arange(D) // GROUP]


def decode_rows(rows: np.ndarray, D: int) -> np.ndarray:
    o, v = decode_parts(rows, D)
    return o + v


def sequence(plane: np.ndarray, table, n: int) -> np.ndarray:
    """Rows [n, H, ...] of a sequence from one plane [NB, BS, H, ...]."""
    BS = plane.shape[1]
    pos = np.arange(n)
    return plane[np.asarray(table)[pos // BS], pos % BS]


def attend(pool: np.ndarray, D: int, q: np.ndarray, tables, lens, scale: float):
    """pool [2, NB, BS, H, row] bytes, q [B, heads, D].

    Returns (out [B, heads, D], weights: list of [H, n] per sequence, bound [B, heads, D], spread [B, heads]): `bound` is
    sum_t p_t (|offset| + |scale (code - 8)| + scale code), `spread` the largest scale * sum_d |q| (|offset| + |scale (code - 8)|) of a
    token, which rounding errors of the weighted sum and of the logits are relative to.
    """
    B, heads, _ = q.shape
    H = pool.shape[3]
    group = heads // H
    out, bound, spread, weights = np.zeros((B, heads, D)), np.zeros((B, heads, D)), np.zeros((B, heads)), []
    for b in range(B):
        n = int(lens[b])
        w = np.zeros((H, n))
        if n:
            ko, kv = decode_parts(sequence(pool[0], tables[b], n), D)
            values = sequence(pool[1], tables[b], n)
            vo, vv = decode_parts(values, D)
            size = np.abs(vo) + np.abs(vv) + code_part(values, D)
            for j in range(heads):
                h = j // group
                l = scale * ((ko[:, h] + kv[:, h]) @ q[b, j])
                spread[b, j] = np.max(abs(scale) * ((np.abs(ko[:, h]) + np.abs(kv[:, h])) @ np.abs(q[b, j])))
                p = np.exp(l - l.max())
                p /= p.sum()
                out[b, j] = p @ (vo[:, h] + vv[:, h])
                bound[b, j] = p @ size[:, h]
                w[h] += p
        weights.append(w)
    return out, weights, bound, spread


def select_tokens(scores: np.ndarray, tables, lens, keep: int, recent: int, sink: int) -> np.ndarray:
    """scores [L, NB, H, BS] -> index [L, B, H, keep]."""
    L, _, H, BS = scores.shape
    index = np.full((L, len(lens), H, keep), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        if n <= keep:
            index[:, b, :, :n] = np.arange(n)
            continue
        pos = np.arange(sink, n - recent)
        blk = np.asarray(tables[b])[pos // BS]
        for l in range(L):
            for h in range(H):
                s = scores[l, blk, h, pos % BS].astype(np.float64)
                s[np.isnan(s)] = -np.inf
                best = pos[np.argsort(-s, kind="stable")[: keep - sink - recent]]
                index[l, b, h] = np.sort(np.concatenate([np.arange(sink), best, np.arange(n - recent, n)]))
    return index


def keep_tokens(pool: np.ndarray, index: np.ndarray, tables, lens, keep: int) -> None:
    """In place on [L, P, NB, BS, H, ...]."""
    BS = pool.shape[3]
    for b, n in enumerate(lens):
        if n <= keep:
            continue
        t = np.asarray(tables[b])
        to = np.arange(keep)
        for l in range(index.shape[0]):
            for h in range(index.shape[2]):
                src = index[l, b, h]
                pool[l][:, t[to // BS], to % BS, h] = pool[l][:, t[src // BS], src % BS, h].copy()
