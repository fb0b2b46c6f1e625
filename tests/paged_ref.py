"""The KV cache in blocks in numpy, from its definitions, in 64 bits: tables, append, read-back, attention.

Block caches: codes [n_blocks, heads, block, dim] int8, scales [n_blocks, heads] float32; a slot is
block id * block + offset, -1 is none.
"""
import numpy as np

from llaisys_amd.hostfmt import bf16_to_f32

# half a step of each type, relative to the value (the kernels round once, to nearest)
HALF_STEP = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float16): 2.0 ** -11, np.dtype(np.uint16): 2.0 ** -8}
# below the normal range a rounding is off by half of the smallest step
TINY = {np.dtype(np.float32): 2.0 ** -150, np.dtype(np.float16): 2.0 ** -25, np.dtype(np.uint16): 2.0 ** -134}


def widen(a):
    """Values of a host array in 64 bits (bf16 comes as uint16 bits)."""
    a = np.asarray(a)
    return bf16_to_f32(a).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


def tables(table, ring, state, old, new, block, rows):
    """(table, ring, state, slots, pos, starts) after a step, or None where it is refused."""
    table, ring, (head, tail), f = table.copy(), ring.copy(), map(int, state), len(ring)
    width = table.shape[1]
    nb = lambda n: -(-int(n) // block)
    slots, pos, starts = np.full(rows, -1, np.int64), np.zeros(rows, np.int64), [0]
    if not (0 <= head <= tail <= head + f) or any(not 0 <= x <= width * block for x in [*old, *new]):
        return None
    back = sum(max(0, nb(o) - nb(n)) for o, n in zip(old, new))
    more = sum(max(0, nb(n) - nb(o)) for o, n in zip(old, new))
    count = sum(max(0, int(n) - int(o)) for o, n in zip(old, new))
    if count > rows or tail + back - head > f or more > tail + back - head:
        return None
    for r, (o, n) in enumerate(zip(old, new)):
        for b in range(nb(n), nb(o)):
            ring[tail % f] = table[r, b]
            tail += 1
    for r, (o, n) in enumerate(zip(old, new)):
        for b in range(nb(o), nb(n)):
            table[r, b] = ring[head % f]
            head += 1
        for p in range(int(o), int(n)):
            t = starts[-1] + p - int(o)
            slots[t], pos[t] = int(table[r, p // block]) * block + p % block, p
        starts.append(starts[-1] + max(0, int(n) - int(o)))
    return table, ring, np.array([head, tail], np.int64), slots, pos, np.array(starts, np.int32)


def append(codes, scales, x, slots):
    """New (codes, scales) of one cache after rows x [rows, heads, dim] went to slots."""
    codes, scales, block = codes.copy(), scales.copy(), codes.shape[2]
    x = widen(x)
    with np.errstate(all="ignore"):
        t = 0
        while t < len(slots):
            if slots[t] < 0:
                t += 1
                continue
            b, first, n = slots[t] // block, slots[t] % block, 1
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] // block == b:
                n += 1
            for h in range(codes.shape[1]):
                run = x[t:t + n, h]
                amax = np.float32(np.nanmax(np.abs(run), initial=0.0, where=~np.isnan(run)))
                was = np.float32(0) if first == 0 else scales[b, h]
                now = max(was, np.float32(amax / np.float32(127)))
                if first and now != was:
                    codes[b, h, :first] = np.rint(codes[b, h, :first].astype(np.float64) * float(was) / float(now))
                q = np.nan_to_num(np.rint(run / np.float64(now)), nan=0.0, posinf=127, neginf=-127)
                codes[b, h, first:first + n] = np.clip(q, -127, 127)
                scales[b, h] = now
            t += n
    return codes, scales


def read(codes, scales, slots):
    """Exact values [rows, heads, dim] of the slots."""
    block = codes.shape[2]
    b, o = slots // block, slots % block
    with np.errstate(all="ignore"):
        return codes[b, :, o].astype(np.float64) * scales[b].astype(np.float64)[:, :, None]


def attend(q, k_codes, k_scale, v_codes, v_scale, table, starts, lens, scale, weight_step):
    """Attention in 64 bits: (out, tol), NaN in `out` at rows that belong to no request.

    tol bounds a kernel's error from the arithmetic alone.  With u = 2^-24 and A = sum p |v| / sum p:
    a score s = sum_c q_c k_c * scale sums dim products in f32, off by at most (dim + 4) u sum |q_c k_c| |scale|,
    and q may enter as two f16 parts, 2^-22 relative; the exponent's argument and the exponential add
    4 u (|s| + |max|) + 4 u.  An error e of every exponent moves a weight by e, and the weighted mean by at most 2 e A.  A weight is rounded to
    weight_step (relative), 2 weight_step A with the sum of weights unrounded; sums of n weights in f32 add 2 n u A.  A weight far
    below the largest, 1, loses more: it enters the product with the values as f16 times 2^11 or more, and the scale of its
    values is at most the one they are summed in, so half of f16's smallest step is 2^-25 2^-11, below 2^-34 of the
    largest weight times a value, for each of the n keys.  Storing rounds once."""
    q_bits, q = np.asarray(q), widen(q)
    block, heads, dim = k_codes.shape[2], k_codes.shape[1], k_codes.shape[3]
    group, u = q.shape[1] // heads, 2.0 ** -24
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for r in range(len(lens)):
        a, e, n = int(starts[r]), int(starts[r + 1]), int(lens[r])
        if e <= a:
            continue
        ids = table[r, :-(-n // block)].astype(np.int64)
        ok = np.repeat((ids >= 0) & (ids < len(k_codes)), block)[:n]
        at = np.where((ids >= 0) & (ids < len(k_codes)), ids, 0)
        seen = np.arange(n)[None, :] <= n - (e - a) + np.arange(e - a)[:, None]
        seen &= ok[None, :]
        for h in range(q.shape[1]):
            kv = []
            for codes, sc in ((k_codes, k_scale), (v_codes, v_scale)):
                x = codes[at, h // group].astype(np.float64) * sc[at, h // group].astype(np.float64)[:, None, None]
                kv.append(x.reshape(-1, dim)[:n])
            k, v = kv
            with np.errstate(all="ignore"):
                s = np.where(seen, (q[a:e, h] @ k.T) * scale, -np.inf)
                size = np.where(seen, (np.abs(q[a:e, h]) @ np.abs(k).T) * abs(scale), 0.0)
                bad = np.isnan(s).any(axis=1, keepdims=True) | (seen @ np.isnan(v) > 0)  # a NaN score, a NaN value that is seen
                s, size, vz = (np.nan_to_num(x, nan=0.0, neginf=-np.inf) for x in (s, size, v))
                top = s.max(axis=1, initial=-np.inf, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isinf(top), 0.0, top)), 0.0)
                total = p.sum(axis=1, keepdims=True)
                o = np.where(total > 0, (p @ vz) / np.where(total > 0, total, 1.0), 0.0)
                spread = np.where(total > 0, (p @ np.abs(vz)) / np.where(total > 0, total, 1.0), 0.0)
                o = np.where(bad, np.nan, o)
            if n:
                sizes = size.max(axis=1, initial=0.0, keepdims=True)
                err = ((dim + 4) * u + 2.0 ** -22) * sizes + 4 * u * (2 * sizes) + 4 * u
                largest = np.where(seen, np.abs(vz).max(axis=1)[None, :], 0.0).max(axis=1, keepdims=True)
                tol[a:e, h] = (2 * err + 2 * weight_step + 2 * n * u) * spread + n * 2.0 ** -34 * largest
                out[a:e, h] = o
            else:
                out[a:e, h] = 0.0
    step = HALF_STEP[q_bits.dtype]
    return out, tol * (1 + step) + step * np.abs(np.nan_to_num(out)) + TINY[q_bits.dtype]
