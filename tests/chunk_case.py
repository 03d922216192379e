"""Definitions in 64 bits (numpy) of the operators of prompts in chunks, and
inputs for them."""
import math

import numpy as np


def chunk_ref(q, start, ks, vs, scale, window=0):
    """q [n][H][hd] float64; start [B + 1]; ks, vs: per sequence [rows][n_kv][hd].
    (out, lse, sum of p |v| of every element); zeros where no sequence has the token."""
    n, H, hd = q.shape
    out, lse, mag = np.zeros((n, H, hd)), np.zeros((n, H)), np.zeros((n, H, hd))
    for b, (k, v) in enumerate(zip(ks, vs)):
        gqa = H // k.shape[1]
        for t in range(start[b], start[b + 1]):
            r = k.shape[0] - (start[b + 1] - t)
            lo = max(0, r + 1 - window) if window else 0
            for h in range(H):
                s = k[lo:r + 1, h // gqa] @ q[t, h] * scale
                e = np.exp(s - s.max())
                p = e / e.sum()
                out[t, h] = p @ v[lo:r + 1, h // gqa]
                mag[t, h] = p @ np.abs(v[lo:r + 1, h // gqa])
                lse[t, h] = s.max() + np.log(e.sum())
    return out, lse, mag


def freqs_ref(n, base, scaling=None, factor=1.0, orig=0, fast=32.0, slow=1.0, factors=None):
    """(radians per position of the n / 2 pairs, magnitude), pair by pair."""
    out, grow = [], 1.0
    for i in range(n // 2):
        f = base ** (-2.0 * i / n)
        if factors is not None:
            f /= float(factors[i])
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            lo = max(0, math.floor(n * math.log(orig / (fast * 2 * math.pi)) / (2 * math.log(base))))
            hi = min(n - 1, math.ceil(n * math.log(orig / (slow * 2 * math.pi)) / (2 * math.log(base))))
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - r) + f / factor * r
            grow = 1 + 0.1 * math.log(factor)
        out.append(f)
    return np.array(out), grow


def turned_ref(x, w, pos, freq, n, interleaved, magnitude, eps):
    """x [n][heads][hd] float64: RMSNorm with w (None: none), then the first n elements turned."""
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    th = pos.astype(np.float64)[:, None, None] * freq
    c, s = np.cos(th) * magnitude, np.sin(th) * magnitude
    y = x.copy()
    first = np.arange(0, n, 2) if interleaved else np.arange(n // 2)
    second = first + 1 if interleaved else first + n // 2
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    assert hd == x.shape[-1]
    return y


class Tables:
    """The host's side of a page table, sequence by sequence as the definition says it."""

    def __init__(self, rng, n_seqs, max_pages, page, n_pages, lens, held):
        self.page, self.max_pages = page, max_pages
        ids = list(rng.permutation(n_pages).astype(int))
        self.lens, self.held = [int(x) for x in lens], [int(x) for x in held]
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        for b in range(n_seqs):
            for i in range(self.held[b]):
                self.table[b, i] = ids.pop()
        self.free = np.full(n_pages, -1, np.int32)
        self.free[:len(ids)] = ids
        self.n_free = len(ids)
        self.next_pos = [int(x) + 7 * b for b, x in enumerate(lens)]

    def plan(self, want, n_tokens):
        """(start, seq, row, pos) of one call; the tables as they are after it."""
        n, page = len(self.lens), self.page
        left, t, target = n_tokens, [], []
        for b in range(n):
            w = min(max(int(want[b]), 0), self.max_pages * page - self.lens[b])
            t.append(min(w, left))
            left -= t[-1]
            target.append(-(-(self.lens[b] + t[-1]) // page))
        for b in range(n):
            for i in range(target[b], self.held[b]):
                self.free[self.n_free] = self.table[b, i]
                self.n_free += 1
            self.held[b] = min(self.held[b], target[b])
        start, seq, row, pos = [0], [], [], []
        top, at = self.n_free, self.n_free
        for b in range(n):
            while self.held[b] < target[b] and at > 0:
                at -= 1
                self.table[b, self.held[b]] = self.free[at]
                self.held[b] += 1
            got = max(0, min(t[b], self.held[b] * page - self.lens[b]))
            seq += [b] * got
            row += list(range(self.lens[b], self.lens[b] + got))
            pos += list(range(self.next_pos[b], self.next_pos[b] + got))
            self.lens[b] += got
            self.next_pos[b] += got
            start.append(start[-1] + got)
        assert top >= at
        self.n_free = at
        pad = n_tokens - start[-1]
        return (np.array(start), np.array(seq + [0] * pad), np.array(row + [-1] * pad), np.array(pos + [0] * pad))
