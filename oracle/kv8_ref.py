"""Plain numpy statements of the paged 8-bit cache (test infrastructure only).

Table kernels as loops, the append in float32 with one rounding per operation (what the kernels compute, so
levels and scales are compared for equality), attention in float64 with a bound on what the kernels may differ by."""
import numpy as np

F32 = np.float32


def extend(tokens, lens, table, free_list, free_count, block_size, max_tokens):
    """Returns (slots, positions, q_start, q_lens, kv_lens, lens, table, free_count)."""
    lens, table = lens.copy(), table.copy()
    width = table.shape[1]
    slots = np.full(max_tokens, -1, np.int32)
    positions = np.full(max_tokens, -1, np.int32)
    q_start, q_lens = [0], []
    asked_blocks = handed = 0
    for r in range(len(lens)):
        n = max(int(tokens[r]), 0)
        at = q_start[-1]
        q_start.append(at + n)
        had = min(max(int(lens[r]), 0), width * block_size)
        lens[r] = had
        held = -(-had // block_size)
        need = -(-(had + n) // block_size) - held
        if had + n > width * block_size or at + n > max_tokens:
            q_lens.append(0)
            continue
        asked_blocks += need
        if need and asked_blocks > free_count:
            q_lens.append(0)
            continue
        for j in range(need):
            table[r, held + j] = free_list[free_count - 1 - handed]
            handed += 1
        for i in range(n):
            p = had + i
            slots[at + i] = table[r, p // block_size] * block_size + p % block_size
            positions[at + i] = p
        lens[r] = had + n
        q_lens.append(n)
    return (slots, positions, np.array(q_start, np.int32), np.array(q_lens, np.int32), lens.copy(), lens, table,
            free_count - handed)


def trim(keep, lens, table, free_list, free_count, block_size):
    """Returns (lens, table, free_list, free_count)."""
    lens, table, free_list = lens.copy(), table.copy(), free_list.copy()
    gone = []
    for r in range(len(lens)):
        stay = min(max(int(keep[r]), 0), int(lens[r]))
        for j in range(-(-stay // block_size), -(-int(lens[r]) // block_size)):
            gone.append(int(table[r, j]))
            table[r, j] = -1
        lens[r] = stay
    for b in reversed(gone):
        free_list[free_count] = b
        free_count += 1
    return lens, table, free_list, free_count


def rotate(x, cos, sin):
    """x [tokens, heads, d] float32; cos, sin [tokens, d / 2]."""
    h = x.shape[-1] // 2
    c, s = cos[:, None].astype(F32), sin[:, None].astype(F32)
    lo, hi = x[..., :h].astype(F32), x[..., h:].astype(F32)
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], axis=-1)


def append(x, levels, scales, slots):
    """x [tokens, heads, d] float32 (rotated) into levels [blocks, heads, size, d] and scales [blocks, heads]."""
    levels, scales = levels.copy(), scales.copy()
    size = levels.shape[2]
    runs = []
    for i, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        if runs and i == runs[-1][-1] + 1 and s % size and slots[i - 1] == s - 1:
            runs[-1].append(i)
        else:
            runs.append([i])
    with np.errstate(all="ignore"):
        for run in runs:
            b, off = divmod(int(slots[run[0]]), size)
            for h in range(levels.shape[1]):
                new = x[run, h].astype(F32)
                old = scales[b, h] if off else F32(0)
                top = np.abs(new).max()
                fresh = F32(top) / F32(127) if np.isfinite(top) else F32(np.nan)
                s = F32(np.nan) if np.isnan(old) or np.isnan(fresh) else max(old, fresh)
                scales[b, h] = s
                if off and s > old > 0:
                    levels[b, h, :off] = np.rint(levels[b, h, :off].astype(F32) * (old / s)).astype(np.int8)
                q = np.clip(np.rint(new / s), -127, 127).astype(np.int8) if s > 0 else 0
                levels[b, h, off:off + len(run)] = q
    return levels, scales


def attention(q, k, v, ks, vs, table, q_start, q_lens, kv_lens, scale, out, max_q=1 << 30):
    """q [tokens, heads, d] float64; returns (out float64, allowed difference before the output's own rounding).

    The allowance per output: probabilities enter the second product as f16, half a step 2^-11 relative to each;
    a score's sum of d products in fp32 is off by at most (d + 4) 2^-23 times the sum of the magnitudes, a
    probability by twice that relative (its own and the normaliser's); exp2 and the remaining fp32 operations stay
    within 2^-19 of the magnitudes.  Probabilities under 2^-29 of the row's largest lose bits: 2^-40 of the largest each."""
    out = out.astype(np.float64).copy()
    slack = np.zeros_like(out)
    size, d = k.shape[2], k.shape[3]
    g = q.shape[1] // k.shape[1]
    for r in range(len(q_lens)):
        length = int(min(max(kv_lens[r], 0), table.shape[1] * size))
        n = int(q_lens[r])
        ids = table[r, :-(-length // size)]
        good = (ids >= 0) & (ids < k.shape[0])
        safe = np.where(good, ids, 0)
        there = np.repeat(good, size)[:length]
        rows = [i for i in range(min(n, max_q)) if 0 <= q_start[r] + i < q.shape[0]]
        if not rows:
            continue
        at = q_start[r] + np.array(rows)
        seen = (np.arange(length)[None] <= (length - n + np.array(rows))[:, None]) & there[None]
        for h in range(q.shape[1]):
            with np.errstate(all="ignore"):
                ksh = np.repeat(ks[safe, h // g].astype(np.float64), size)[:length]
                vsh = np.repeat(vs[safe, h // g].astype(np.float64), size)[:length]
                kk = k[safe, h // g].reshape(-1, d)[:length].astype(np.float64)
                vv = v[safe, h // g].reshape(-1, d)[:length].astype(np.float64)
                s = (q[at, h] @ kk.T) * ksh * scale
                mag = (np.abs(q[at, h]) @ np.abs(kk).T) * np.abs(ksh) * scale
                s = np.where(seen, s, -np.inf)
                top = s.max(axis=1, initial=-np.inf, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isneginf(top), 0, top)), 0)
                total = p.sum(axis=1, keepdims=True)
                w = np.where(p > 0, p, 0) if not np.isnan(p).any() else p
                val = np.where(seen[:, :, None], vv[None] * vsh[None, :, None], 0) if np.isnan(vsh).any() else None
                if val is None:
                    o, a = w @ (vv * vsh[:, None]), w @ np.abs(vv * vsh[:, None])
                else:
                    o, a = np.einsum("ij,ijd->id", w, val), np.einsum("ij,ijd->id", w, np.abs(val))
                o = np.where(total == 0, 0, o / np.where(total == 0, 1, total))
                a = np.where(total == 0, 0, a / np.where(total == 0, 1, total))
                delta = np.where(seen, mag, 0).max(axis=1, initial=0, keepdims=True) * (d + 4) * 2.0 ** -23
                big = np.where(seen[:, :, None], np.abs(vv * vsh[:, None])[None], 0).max(axis=1, initial=0) \
                    if np.isfinite(vsh).all() else 0
                tiny = length * 2.0 ** -40 * big / np.where(total == 0, 1, total)
            out[at, h] = o
            slack[at, h] = a * (2.0 ** -11 + 2 * delta + 2.0 ** -19) + tiny
    return out, slack
