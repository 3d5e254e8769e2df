"""The 4-bit paged cache and the step's block tables in numpy, in 64 bits and from the definitions:
the oracle of the operators in `vllm_ttkv.ops` (`q4_*`, `plan_step`, `release_blocks`)."""
import numpy as np

LIMIT = 57344.0


def quantise(x, g):
    """x [..., d] -> (codes int [..., d], scale fp16 [..., d/g], minimum fp16 [..., d/g])."""
    x = np.asarray(x, np.float64)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // g, g)
    bad = ~np.isfinite(x).all(-1)
    x = np.clip(np.where(bad[..., None], 0.0, x), -LIMIT, LIMIT)
    lo, hi = x.min(-1), x.max(-1)
    m = (lo + 0.0).astype(np.float16)                 # -0 is stored as 0
    s = ((hi - lo) / 15.0).astype(np.float16)
    sd = s.astype(np.float64)[..., None]
    c = np.rint((x - m.astype(np.float64)[..., None]) / np.where(sd > 0, sd, 1.0))
    c = np.where(sd > 0, np.clip(c, 0, 15), 0).astype(np.int64)
    s = np.where(bad, np.float16(np.nan), s)
    m = np.where(bad, np.float16(0), m)
    return c.reshape(*c.shape[:-2], c.shape[-2] * g), s, m


def values(c, s, m):
    """The values that codes stand for, in 64 bits."""
    g = c.shape[-1] // s.shape[-1]
    return m.astype(np.float64).repeat(g, -1) + s.astype(np.float64).repeat(g, -1) * c


def panel_bytes(d, g):
    return 16 * (d + 8 * d // g)


def put(cache, slot, h, block_size, kq, vq):
    """Store one token's (codes, scale, minimum) of K and of V of head h into a uint8 cache, byte by byte."""
    d = kq[0].shape[-1]
    ng = kq[1].shape[-1]
    blk, off = divmod(int(slot), block_size)
    pan = cache[blk, h, off // 16]
    o = off % 16

    def nib(byte, lane, code):
        keep = 0xF0 if lane % 2 == 0 else 0x0F
        pan[byte] = (int(pan[byte]) & keep) | (int(code) << (4 * (lane % 2)))

    for lane in range(d):
        nib(o * (d // 2) + (lane % 32) // 8 * (d // 8) + lane // 32 * 4 + lane % 8 // 2, lane, kq[0][lane])
        nib(8 * d + o // 2 * d + (lane % 32) // 4 * (d // 8) + lane // 32 * 4 + o % 2 * 2 + lane % 4 // 2, lane, vq[0][lane])
    for base, (_, s, m) in ((16 * d, kq), (16 * d + 64 * ng, vq)):
        for i in range(ng):
            at = base + (o * ng + i) * 4
            pan[at:at + 2] = np.frombuffer(np.float16(s[i]).tobytes(), np.uint8)
            pan[at + 2:at + 4] = np.frombuffer(np.float16(m[i]).tobytes(), np.uint8)


def attend(q, K, V, scale, G):
    """Causal attention of the last q tokens of a sequence: q [nq, HQ, d] over K, V [n, H, d] (64 bits)."""
    nq, HQ, d = q.shape
    n = K.shape[0]
    out = np.zeros((nq, HQ, d))
    for h in range(HQ):
        s = q[:, h] @ K[:, h // G].T * scale
        s[np.arange(n)[None] > (n - nq + np.arange(nq))[:, None]] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = p @ V[:, h // G] / p.sum(-1, keepdims=True)
    return out


def plan(table, seq, qsl, free, count, block_size, n_tokens):
    """One step's plan, request by request: (table, slots, positions, count, refused rows)."""
    table, free = table.copy(), list(free[:count])
    slots, pos = np.full(n_tokens, -1, np.int64), np.zeros(n_tokens, np.int64)
    refused, dry = [], False
    for r in range(len(seq)):
        a, b = int(qsl[r]), int(qsl[r + 1])
        n, new = int(seq[r]), b - a
        held, want = -(-(n - max(new, 0)) // block_size), -(-n // block_size)
        held = max(held, 0)
        bad = a < 0 or new < 0 or b > n_tokens or n < new or want > table.shape[1]
        if not bad and want > held and (dry or want - held > len(free)):
            bad = dry = True
        if bad:
            refused.append(r)
            end = 1 if new > n else max(want, held + 1)
            table[r, held:end] = -1
            continue
        for i in range(held, want):
            table[r, i] = free.pop()
        for t in range(a, b):
            p = n - new + t - a
            pos[t] = p
            slots[t] = int(table[r, p // block_size]) * block_size + p % block_size
    return table, slots, pos, len(free), refused


def release(table, lens, free, count, block_size):
    """The free list after the blocks of `lens` tokens of each row have been returned: (list, refused rows)."""
    out, refused, full = list(free[:count]), [], False
    for r, n in enumerate(lens):
        ids = [int(x) for x in table[r, :max(0, -(-int(n) // block_size))]]
        if -(-int(n) // block_size) > table.shape[1] or min(ids, default=0) < 0:
            refused.append(r)
        elif ids and (full or len(out) + len(ids) > len(free)):
            full = True
            refused.append(r)
        else:
            out += ids
    return out, refused
