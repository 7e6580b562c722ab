"""The 8-bit cache and the verification of drafts from their definitions, in 64 bits and one row at a time (numpy)."""
import math

import numpy as np
import torch

# what the codes 0..126 stand for: 1 sign, 4 exponent and 3 mantissa bits
NUMBERS = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127])


def encode(x):
    """Codes (uint8) and scale bytes of rows [..., d]; a row whose numbers are not all finite in 32 bits: codes 0, byte 255."""
    x = np.asarray(x, dtype=np.float64)
    flat = x.reshape(-1, x.shape[-1])
    codes, bytes_ = np.zeros(flat.shape, np.uint8), np.zeros(flat.shape[0], np.uint8)
    for r, row in enumerate(flat):
        with np.errstate(over="ignore"):
            finite = np.isfinite(row.astype(np.float32)).all()
        if not finite:
            bytes_[r] = 255
            continue
        top = np.abs(row).max()
        power = 0
        if top > 0:
            power = -110
            while top > 448.0 * 2.0 ** power:
                power += 1
        y = np.abs(row) / 2.0 ** power
        up = np.clip(np.searchsorted(NUMBERS, y), 1, 126)
        below, above = NUMBERS[up - 1], NUMBERS[up]
        higher = (above - y < y - below) | ((above - y == y - below) & (up % 2 == 0))
        codes[r] = np.where(higher, up, up - 1) | np.where(np.signbit(row), 128, 0)
        bytes_[r] = power + 127
    return codes.reshape(x.shape), bytes_.reshape(x.shape[:-1])


def decode(codes, bytes_):
    """Numbers of codes [..., d] with scale bytes [...]; NaN for byte 255."""
    codes, bytes_ = np.asarray(codes), np.asarray(bytes_).astype(np.int64)
    value = NUMBERS[np.minimum(codes & 127, 126)] * np.where(codes & 128, -1.0, 1.0)
    scale = np.where(bytes_ == 255, np.nan, np.ldexp(1.0, bytes_ - 127))
    return value * scale[..., None]


def random_pages(ops, rng, num_pages, n_kv, page_size, d, spread=1.0, device="cuda"):
    """Pages full of rows of the kind that a store leaves, made on the host."""
    rows = rng.standard_normal((2, num_pages, n_kv, page_size, d)) * np.exp(spread * rng.standard_normal((2, num_pages, n_kv, page_size, 1)))
    (kc, kb), (vc, vb) = encode(rows[0]), encode(rows[1])
    return ops.QuantPages(torch.from_numpy(kc).to(device).view(torch.float8_e4m3fn), torch.from_numpy(vc).to(device).view(torch.float8_e4m3fn),
                          torch.from_numpy(kb).to(device), torch.from_numpy(vb).to(device))


class Batch:
    """A step's requests over shuffled pages: rows and cached lengths of each, block tables and starts on the device."""

    def __init__(self, rng, rows, past, page_size, lengths=None, spare=2, width=0, device="cuda"):
        self.rows, self.past = list(rows), list(past)
        self.held = list(lengths) if lengths is not None else [r + p for r, p in zip(rows, past)]
        blocks = [-(-n // page_size) for n in self.held]
        self.num_pages = sum(blocks) + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((len(self.rows), max(blocks + [1]) + width), -1, np.int32)
        at = 0
        for b, n in enumerate(blocks):
            self.table[b, :n] = order[at: at + n]
            at += n
        self.starts = np.concatenate(([0], np.cumsum(self.rows))).astype(np.int32)
        self.tokens, self.page_size, self.device = int(self.starts[-1]), page_size, device

    def args(self):
        to = lambda x: torch.tensor(np.asarray(x, np.int32), device=self.device)  # noqa: E731
        return (to(self.starts), to(self.held), to(self.past), to(self.table), len(self.rows), self.rows, max(self.held + [0]))


def first_key(pos, window):
    if window > 0:
        return max(0, pos - window + 1)
    if window < 0:
        return pos // -window * -window
    return 0


def attention(q, pages, batch, n_q, n_kv, d, window, scale, codes_of_p):
    """(out, bound) in 64 bits: the definition, and how far a kernel may be from it.

    The bound counts, per entry of a row, with w_j = |p_j v_j| / sum p:
      * the score.  Its error is at most (d + 4) 2^-23 of sum_i |q_i k_i| for 32-bit sums of exact products; with `codes_of_p`, q's
        two codes miss at most 2^-10 where q's largest is 224 or more: 2^-17 max|q| sum_i |k_i|.  Twice that (this key's and
        the denominator's) times w_j.
      * p.  An exponential's own error, under 2^-20, and with `codes_of_p` the two codes': 2^-8 of p, or 2^-10 where the tile's
        largest p 2^e is 2^8 up to a factor that rounds: 2^-17 of the largest p_i scale_i of the tile of 128 keys, times |code_j|.
      * the 32-bit sums over the keys: n 2^-23 of sum_j w_j.
    The rounding of the result to its type is the caller's."""
    value = lambda codes, bytes_: decode(codes.view(torch.uint8).cpu().numpy(), bytes_.cpu().numpy())  # noqa: E731
    k, v = value(pages.k, pages.k_scale), value(pages.v, pages.v_scale)
    v_scale = np.where(pages.v_scale.cpu().numpy() == 255, np.nan, np.ldexp(1.0, pages.v_scale.cpu().numpy().astype(np.int64) - 127))
    q = q.double().cpu().numpy().reshape(-1, n_q, d)
    out, bound = np.zeros((batch.tokens, n_q, d)), np.zeros((batch.tokens, n_q, d))
    for b, rows in enumerate(batch.rows):
        n, ps = batch.held[b], batch.page_size
        if n == 0:
            continue
        own = batch.table[b, : -(-n // ps)]
        for kvh in range(n_kv):
            keys, values, scales = (x[own, kvh].reshape((-1,) + x.shape[3:])[:n] for x in (k, v, v_scale))
            for i in range(rows):
                pos, t = batch.past[b] + i, batch.starts[b] + i
                lo, hi = first_key(pos, window), min(pos, n - 1)
                if hi < lo:
                    continue
                kk, vv, ss = keys[lo: hi + 1], values[lo: hi + 1], scales[lo: hi + 1]
                heads = slice(kvh * (n_q // n_kv), (kvh + 1) * (n_q // n_kv))
                qq = q[t, heads]
                s = qq @ kk.T * scale
                with np.errstate(invalid="ignore"):
                    p = np.exp(s - np.nanmax(s, axis=-1, keepdims=True))
                total = p.sum(axis=-1, keepdims=True)
                p /= total
                out[t, heads] = p @ vv
                miss = (d + 4) * 2.0 ** -23 * (np.abs(qq) @ np.abs(kk).T) * scale
                if codes_of_p:
                    miss += 2.0 ** -17 * np.abs(qq).max(axis=-1, keepdims=True) * np.abs(kk).sum(axis=-1) * scale
                w = p * (2 * miss.max(axis=-1, keepdims=True) + 2.0 ** -20 + len(kk) * 2.0 ** -23 + (2.0 ** -8 if codes_of_p else 0.0))
                bound[t, heads] = w @ np.abs(vv)
                if codes_of_p:
                    tile = np.arange(lo, hi + 1) // 128
                    for one in np.unique(tile):
                        at = tile == one
                        bound[t, heads] += 2.0 ** -17 * (p[:, at] * ss[at]).max(axis=-1, keepdims=True) * np.abs(vv[at] / ss[at][:, None]).sum(axis=0)
    return out.reshape(batch.tokens, -1), bound.reshape(batch.tokens, -1)


def mix32(x):
    x &= 0xFFFFFFFF
    x ^= x >> 16
    x = x * 0x7FEB352D & 0xFFFFFFFF
    x ^= x >> 15
    x = x * 0x846CA68B & 0xFFFFFFFF
    return x ^ x >> 16


def uniform(h):
    return ((h >> 9) + 0.5) / 8388608.0


def mix32_all(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xFFFFFFFF)
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        x ^= x >> np.uint64(shift)
        x = x * np.uint64(factor) & np.uint64(0xFFFFFFFF)
    return x ^ x >> np.uint64(16)


def verify(logits, drafts, starts, draft_probs, temperature, seeds, positions):
    """(tokens, counts, gap): the definition in 64 bits, and the least relative distance between two numbers that a decision compared."""
    logits = np.asarray(logits, np.float64)
    vocab, gap = logits.shape[1], math.inf
    tokens, counts = np.full(len(logits), -1, np.int64), np.zeros(len(starts) - 1, np.int64)
    for b in range(len(starts) - 1):
        rows = range(starts[b], starts[b + 1])
        t = 0.0 if temperature is None else float(temperature[b])
        for i, row in enumerate(rows):
            counts[b] = i + 1
            last, x = row == starts[b + 1] - 1, int(drafts[row])
            if t == 0.0:
                best = int(np.nanargmax(logits[row]))
                if not last and x == best:
                    tokens[row] = x
                    continue
                tokens[row] = best
                break
            e = np.exp((logits[row] - np.nanmax(logits[row])) / t)
            p = e / np.nansum(e)
            key = mix32(mix32((int(seeds[b]) & 0xFFFFFFFF) ^ 0x9E3779B9) ^ (int(positions[b]) + i))
            if not last and 0 <= x < vocab:
                q = 1.0 if draft_probs is None else float(draft_probs[row, x])
                u = uniform(mix32(key ^ 0xFFFFFFFF))
                gap = min(gap, abs(u * q - p[x]) / max(p[x], u * q))
                if u * q < p[x]:
                    tokens[row] = x
                    continue
            w = p.copy()
            if not last:
                if draft_probs is not None:
                    w = np.maximum(p - np.asarray(draft_probs[row], np.float64), 0.0)
                elif 0 <= x < vocab:
                    w[x] = 0.0
            if not np.nanmax(w) > 0:
                w = p
            rate = w / -np.log(uniform(mix32_all(key + np.arange(vocab, dtype=np.uint64) * np.uint64(0x85EBCA6B))))
            order = np.argsort(np.where(np.isnan(rate), -1.0, rate))
            tokens[row] = order[-1]
            if vocab > 1:
                gap = min(gap, 1 - rate[order[-2]] / rate[order[-1]])
            break
    return tokens, counts, gap
