"""The operators of the 4-bit paged cache and of the step's block tables, as cases to measure.

Each case runs in a plain form (elementary torch operations) or, with `own` true, through the
framework's entry points (`vllm_ttkv.ops`). Kinds of case:

* store:   `q4_write_paged` quantises a step's keys and values into the paged cache, then
           `q4_read_paged` reads the same slots back as the values they stand for.
* decode:  `q4_decode_paged`, one query token per request over its stored tokens.
* prefill: `q4_prefill_paged`, a chunk of query tokens per request, causal over its stored tokens.
* plan:    `release_blocks` returns finished requests' blocks to the free list, then `plan_step`
           extends the block tables of the running ones and maps the step's tokens to slots.

The cache: uint8 [blocks, H, block_size / 16, panel bytes]. A panel holds 16 tokens of one KV head:
K codes (8 d bytes), V codes (8 d bytes), then (scale, minimum) as two fp16 per token and group of
lanes, for K and for V. A code c of a group stands for minimum + scale * c.
"""
import pathlib
import sys

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LIMIT = 57344.0            # values beyond it are stored as it
DEV = "cuda"


def listed():
    """Heads, lengths and block size of the repository's benchmark where it has them (24 query and 8
    KV heads of 128, 4322, 7379, 14402 and 16384 tokens, blocks of 16), else generic ones."""
    return [
        # one decode step's tokens of a small batch: latency
        dict(name="store step of 8", kind="store", tokens=8, H=8, d=128, group=128, block=16, dtype="bf16", pad=0),
        # a ragged first chunk in fp32 with small groups, an odd count and padding slots at its end
        dict(name="store odd chunk", kind="store", tokens=1081, H=4, d=64, group=32, block=32, dtype="fp32", pad=7),
        # a long prompt's keys and values: bandwidth
        dict(name="store prompt", kind="store", tokens=16384, H=8, d=128, group=64, block=16, dtype="bf16", pad=0),
        # one short request: latency
        dict(name="decode one short", kind="decode", reqs=1, lo=257, hi=257, HQ=32, H=8, d=64, group=64, block=16, dtype="fp16"),
        # the benchmark's decode step
        dict(name="decode batch", kind="decode", reqs=8, lo=4322, hi=4322, HQ=24, H=8, d=128, group=128, block=16, dtype="bf16"),
        # one very long request on few heads (a shard of a model): the split over the tokens
        dict(name="decode long", kind="decode", reqs=1, lo=131071, hi=131071, HQ=16, H=2, d=128, group=32, block=64, dtype="fp16"),
        # the sweep's largest batch, ragged
        dict(name="decode ragged", kind="decode", reqs=64, lo=1, hi=14402, HQ=24, H=8, d=128, group=128, block=16, dtype="bf16"),
        # a few drafted tokens per request, checked at once
        dict(name="prefill few", kind="prefill", reqs=16, q_lo=1, q_hi=5, lo=33, hi=4322, HQ=32, H=8, d=64, group=32, block=32, dtype="fp16"),
        # the benchmark's chunk
        dict(name="prefill chunk", kind="prefill", reqs=8, q_lo=256, q_hi=256, lo=7379, hi=7379, HQ=24, H=8, d=128, group=128, block=16, dtype="bf16"),
        # long chunks of two long requests, ragged
        dict(name="prefill long", kind="prefill", reqs=2, q_lo=1024, q_hi=2048, lo=8192, hi=16384, HQ=32, H=8, d=128, group=64, block=64, dtype="bf16"),
        # a decode step's tables
        dict(name="plan decode", kind="plan", reqs=64, q_lo=1, q_hi=1, lo=1, hi=14402, done=3, block=16, pad=0),
        # prompts and decodes mixed in a large batch, padded to a captured size
        dict(name="plan mixed", kind="plan", reqs=512, q_lo=1, q_hi=64, lo=1, hi=8192, done=40, block=16, pad=300),
    ]


def _log(rng, a, b):
    return int(round(a * (b / a) ** rng.random())) if b > a else a


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill", "plan"])
    if kind == "plan":
        q_hi = _log(rng, 1, 128)
        reqs = _log(rng, 1, 1024)
        return dict(kind=kind, reqs=reqs, q_lo=1, q_hi=q_hi, lo=1, hi=_log(rng, max(q_hi, 16), 14402), done=rng.randint(0, reqs // 2),
                    block=rng.choice([16, 32, 64]), pad=rng.randint(0, 64))
    d = rng.choice([64, 128])
    base = dict(kind=kind, H=rng.choice([1, 2, 4, 8]), d=d, group=rng.choice([g for g in (32, 64, 128) if g <= d]),
                block=rng.choice([16, 32, 64]))
    if kind == "store":
        return dict(base, tokens=_log(rng, 1, 16384), dtype=rng.choice(["bf16", "fp16", "fp32"]), pad=rng.choice([0, 0, 5]))
    G = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    base = dict(base, HQ=base["H"] * G, dtype=rng.choice(["bf16", "fp16"]))
    if kind == "decode":
        reqs = _log(rng, 1, 64)
        hi = _log(rng, 1, min(65536, 393216 // reqs))
        return dict(base, reqs=reqs, lo=rng.choice([1, max(1, hi // 2), hi]), hi=hi)
    reqs = _log(rng, 1, 16)
    q_hi = _log(rng, 1, min(2048, 4096 // (reqs * max(1, base["HQ"] // 16))))
    hi = max(q_hi, _log(rng, 1, min(16384, 65536 // reqs)))
    return dict(base, reqs=reqs, q_lo=rng.randint(1, q_hi), q_hi=q_hi, lo=q_hi, hi=hi)


# ------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """(seq_lens, query lengths, whether finished) of a case: lengths of the case's own in the order
    that the seed gives. The longest is always among them."""
    n = case["reqs"]
    r = np.random.default_rng([n, case["lo"], case["hi"], case["block"]])
    seq = r.integers(case["lo"], case["hi"] + 1, n)
    seq[0] = case["hi"]
    ql = r.integers(case["q_lo"], case["q_hi"] + 1, n) if "q_lo" in case else np.ones(n, np.int64)
    order = np.random.default_rng(seed).permutation(n)
    return seq[order], np.minimum(ql, seq)[order], (np.arange(n) >= n - case.get("done", 0))[order]


def _int32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device=DEV)


def _paged_store(case, seq, gen, seed):
    """A cache filled with quantised tokens and the requests' block table (blocks in random order).
    Keys carry a few channels of larger size, as keys do."""
    H, d, g, bs = case["H"], case["d"], case["group"], case["block"]
    nb = -(-seq // bs)
    total = int(nb.sum()) + 3
    perm = np.random.default_rng(seed + 1).permutation(total)
    table = np.zeros((len(seq), int(nb.max()) + 1), np.int64)
    at = 0
    for r, n in enumerate(nb):
        table[r, :n] = perm[at:at + n]
        at += n
    cache = torch.empty(total, H, bs // 16, 16 * (d + 8 * d // g), dtype=torch.uint8, device=DEV)
    boost = torch.ones(H, 1, d, device=DEV)
    boost[:, :, torch.randperm(d, generator=gen, device=DEV)[:4]] = 8.0
    step = max(1, (1 << 25) // (H * bs * d))
    for b in range(0, total, step):
        n = min(step, total - b)
        k = torch.randn(n, H, bs, d, generator=gen, device=DEV) * boost
        v = torch.randn(n, H, bs, d, generator=gen, device=DEV)
        rows = [_quantise(x.view(n, H, bs // 16, 16, d), g) for x in (k, v)]
        cache[b:b + n] = _panels(rows[0], rows[1])
    return cache, _int32(table)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "plan":
        return _prepare_plan(s, seed)
    H, d, bs, dt = case["H"], case["d"], case["block"], DT[case["dtype"]]
    if case["kind"] == "store":
        n, pad = case["tokens"], case["pad"]
        blocks = -(-n // bs) + 2
        # requests own whole blocks in any order; tokens are consecutive within them
        perm = np.random.default_rng(seed).permutation(blocks)
        t = np.arange(n)
        slots = np.concatenate([perm[t // bs] * bs + t % bs, np.full(pad, -1)])
        s["slots"] = torch.as_tensor(slots, dtype=torch.int64, device=DEV)
        k = torch.randn(n + pad, H, d, generator=gen, device=DEV)
        k[:, :, torch.randperm(d, generator=gen, device=DEV)[:4]] *= 8.0
        s["k"], s["v"] = k.to(dt), torch.randn(n + pad, H, d, generator=gen, device=DEV).to(dt)
        s["cache"] = torch.zeros(blocks, H, bs // 16, 16 * (d + 8 * d // case["group"]), dtype=torch.uint8, device=DEV)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    seq, ql, _ = _lengths(case, seed)
    s["cache"], s["table"] = _paged_store(case, seq, gen, seed)
    s["seq"], s["q_len"] = _int32(seq), _int32(ql)
    s["q_start"] = _int32(np.cumsum(ql) - ql)
    s["max_q"], s["max_seq"] = int(ql.max()), int(seq.max())
    s["q"] = torch.randn(int(ql.sum()), case["HQ"], d, generator=gen, device=DEV).to(dt)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = d ** -0.5
    return s


def _prepare_plan(s, seed):
    r = np.random.default_rng(seed)
    bs, n = s["block"], s["reqs"]
    seq, ql, gone = _lengths(s, seed)
    fin = np.where(gone, seq, 0)                    # lengths of the requests that have finished
    seq, ql = np.where(gone, 0, seq), np.where(gone, 0, ql)
    held = np.where(fin > 0, -(-fin // bs), -(-(seq - ql) // bs))
    need = -(-seq // bs) - np.where(fin > 0, 0, held)
    cols = max(int(held.max()), int((-(-seq // bs)).max())) + 2
    spare = int(need.sum()) + 5
    total = int(held.sum()) + spare
    perm = r.permutation(total)
    table = np.full((n, cols), -1, np.int64)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = perm[at:at + h]
        at += h
    free = np.zeros(total, np.int64)
    free[:spare] = perm[at:]
    tokens = int(ql.sum()) + s["pad"]
    s["table"], s["seq"], s["done_lens"] = _int32(table), _int32(seq), _int32(fin)
    s["qsl"] = _int32(np.concatenate([[0], np.cumsum(ql)]))
    s["free"], s["count"] = _int32(free), _int32([spare])
    s["count1"], s["count2"] = _int32([0]), _int32([0])
    s["slots"] = torch.zeros(tokens, dtype=torch.int64, device=DEV)
    s["positions"] = torch.zeros(tokens, dtype=torch.int64, device=DEV)
    return s


# ------------------------------------------------------------------ the plain forms
def _to_half(x):
    """fp64 >= 0 rounded once to fp16 (a direct cast goes through fp32 and may round twice)."""
    step = torch.exp2(torch.frexp(x).exponent.clamp(min=-13).double() - 11)
    return ((x / step).round() * step).half()


def _quantise(x, g):
    """(codes uint8 [..., d], scale and minimum fp16 [..., d/g, 2]) of x [..., d]."""
    x = x.float().unflatten(-1, (-1, g))
    bad = ~torch.isfinite(x).all(-1)
    x = x.clamp(-LIMIT, LIMIT)
    lo, hi = x.amin(-1), x.amax(-1)
    m = lo.half()
    # the scale's rounding and which code is nearest are settled in 64 bits: values lie next to the
    # border between two
    s = _to_half((hi.double() - lo.double()) / 15.0)
    t = (x.double() - m.double().unsqueeze(-1)) / s.double().unsqueeze(-1)
    c = torch.where(s.unsqueeze(-1) > 0, t.round().clamp(0, 15), 0.0)
    c = torch.where(bad.unsqueeze(-1), 0.0, c).to(torch.uint8)
    meta = torch.stack([torch.where(bad, float("nan"), s), torch.where(bad, 0.0, m)], -1)
    return c.flatten(-2), meta


def _k_bytes(c):
    """K code bytes of a token [..., d/2]: chunk a of four holds lanes 32 w + 8 a + (0..7) for each w."""
    c = c.unflatten(-1, (-1, 4, 4, 2)).transpose(-4, -3)
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-3)


def _v_bytes(c):
    """V code bytes of a token [..., 8, d/32, 2]: lanes 32 j + 4 b + (0..3) for each b and j."""
    c = c.unflatten(-1, (-1, 8, 2, 2)).transpose(-4, -3)
    return c[..., 0] | (c[..., 1] << 4)


def _panels(k, v):
    """Whole panels [..., panel bytes] of the (codes, meta) of 16 tokens each."""
    kb = _k_bytes(k[0]).flatten(-2)
    vb = _v_bytes(v[0])                                            # [..., 16, 8, d/32, 2]
    vb = vb.unflatten(-4, (8, 2)).movedim(-4, -2).flatten(-5)      # pairs of tokens next to each other
    return torch.cat([kb, vb, k[1].contiguous().view(torch.uint8).flatten(-3), v[1].contiguous().view(torch.uint8).flatten(-3)], -1)


def _fields(cache, d, g):
    """Views of a cache's four fields, a token's place as two indexes (pair of tokens, which of them)."""
    k = cache[..., :8 * d].unflatten(-1, (8, 2, d // 2))
    v = cache[..., 8 * d:16 * d].unflatten(-1, (8, 8, d // 32, 2, 2))
    n = 64 * (d // g)
    mk = cache[..., 16 * d:16 * d + n].unflatten(-1, (8, 2, d // g, 4))
    mv = cache[..., 16 * d + n:].unflatten(-1, (8, 2, d // g, 4))
    return k, v, mk, mv


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1)


def _values(kb, vb, mk, mv, d, g):
    """K and V values [..., d] fp32 of a token's bytes (`_k_bytes`, `_v_bytes`) and meta bytes."""
    ck = _nibbles(kb.unflatten(-1, (4, d // 32, 4))).transpose(-4, -3).flatten(-4)
    cv = _nibbles(vb).transpose(-4, -3).flatten(-4)
    out = []
    for c, meta in ((ck, mk), (cv, mv)):
        sm = meta.contiguous().view(torch.float16).float()
        out.append((c.unflatten(-1, (-1, g)).float() * sm[..., :1] + sm[..., 1:]).flatten(-2))
    return out


def _plain_store(s):
    d, g, bs, H = s["d"], s["group"], s["block"], s["H"]
    keep = s["slots"] >= 0
    slots = torch.where(keep, s["slots"], 0)
    blk, off = slots // bs, slots % bs
    pan, pair, par = off // 16, (off % 16) // 2, off % 2
    k, v, mk, mv = _fields(s["cache"], d, g)
    (ck, sk), (cv, sv) = _quantise(s["k"], g), _quantise(s["v"], g)
    at = tuple(x[keep] for x in (blk, pan, pair, par))
    h = torch.arange(H, device=DEV)

    def put(field, x):
        field[at[0][:, None], h, at[1][:, None], at[2][:, None], at[3][:, None]] = x[keep]

    put(k, _k_bytes(ck))
    put(mk, sk.contiguous().view(torch.uint8))
    put(mv, sv.contiguous().view(torch.uint8))
    vt = v.movedim(-2, -4)                                         # [..., pair, which, 8, d/32, 2]
    put(vt, _v_bytes(cv))
    i = (blk[:, None], h, pan[:, None], pair[:, None], par[:, None])
    kk, vv = _values(k[i], vt[i], mk[i], mv[i], d, g)
    keep = keep[:, None, None]
    return {"k": torch.where(keep, kk.to(s["k"].dtype), 0), "v": torch.where(keep, vv.to(s["v"].dtype), 0)}


def _plain_attend(s):
    """Chunks padded to the longest, queries [B, Q, HQ, d], stored tokens [B, n, H, d]."""
    d, g, bs, H, B = s["d"], s["group"], s["block"], s["H"], s["reqs"]
    Q, n, G = s["max_q"], s["max_seq"], s["HQ"] // s["H"]
    blocks = -(-n // bs)
    seq, ql = s["seq"].long(), s["q_len"].long()
    t = torch.arange(blocks * bs, device=DEV)
    tab = torch.where(t[::bs] < seq[:, None], s["table"][:, :blocks].long(), 0)
    k, v, mk, mv = _fields(s["cache"][tab], d, g)                  # [B, blocks, H, panels, pair, which, ...]
    v = v.movedim(-2, -4)
    k, v, mk, mv = (x.movedim(2, 1).flatten(2, 5) for x in (k, v, mk, mv))      # [B, H, n, ...]
    kk, vv = _values(k, v, mk, mv, d, g)
    j = torch.arange(Q, device=DEV)
    rows = (s["q_start"].long()[:, None] + j).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, d)
    sc = (q @ kk.transpose(-1, -2) * s["scale"]).unflatten(2, (Q, G))
    seen = t < (seq[:, None] - ql[:, None] + j + 1).clamp(max=seq[:, None])[..., None]        # [B, Q, n]
    seen = seen[:, None, :, None]
    sc = torch.where(seen, sc, float("-inf"))
    p = torch.where(seen, (sc - sc.amax(-1, keepdim=True)).exp(), 0.0)
    vv = torch.where((t < seq[:, None])[:, None, :, None], vv, 0.0)
    o = (p.flatten(2, 3) @ vv).unflatten(2, (Q, G)) / p.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).flatten(2, 3)[j < ql[:, None]]
    return o.to(s["q"].dtype)


def _plain_plan(s):
    bs = s["block"]
    table, free, seq = s["table"], s["free"], s["seq"].long()
    # the finished requests' blocks onto the free list, request by request
    back = (s["done_lens"].long() + bs - 1) // bs
    c = torch.arange(table.shape[1], device=DEV)
    ids = table[c < back[:, None]]
    count = s["count"].long()
    free[(count + torch.arange(ids.numel(), device=DEV))] = ids
    count1 = count + ids.numel()
    # the running requests' new blocks off its end
    qsl = s["qsl"].long()
    ql = qsl[1:] - qsl[:-1]
    held, want = (seq - ql + bs - 1) // bs, (seq + bs - 1) // bs
    end = (want - held).cumsum(0)
    first = end - (want - held)
    fresh = (c >= held[:, None]) & (c < want[:, None])
    take = (count1 - 1 - (first[:, None] + c - held[:, None])).clamp(min=0)
    table.copy_(torch.where(fresh, free[take], table))
    t = torch.arange(s["slots"].numel(), device=DEV)
    r = torch.searchsorted(qsl[1:], t, right=True).clamp(max=seq.numel() - 1)
    pos = seq[r] - ql[r] + t - qsl[r]
    real = t < qsl[-1]
    pos = torch.where(real, pos, 0)
    slots = torch.where(real, table[r, pos // bs].long() * bs + pos % bs, -1)
    return {"table": table, "slots": slots, "positions": pos, "free": free, "count": (count1 - end[-1]).to(torch.int32)}


# ------------------------------------------------------------------ the framework's calls
def _framework():
    root = str(pathlib.Path(__file__).resolve().parents[1] / "ttkv-vllm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from vllm_ttkv import ops
    from vllm_ttkv.q4 import Q4Layout
    return ops, Q4Layout


def _own_run(s):
    ops, Q4Layout = _framework()
    if s["kind"] == "plan":
        ops.release_blocks(s["table"], s["done_lens"], s["free"], s["count"], s["block"], free_count_out=s["count1"])
        ops.plan_step(s["table"], s["seq"], s["qsl"], s["free"], s["count1"], s["block"], s["slots"],
                      positions=s["positions"], free_count_out=s["count2"])
        return {"table": s["table"], "slots": s["slots"], "positions": s["positions"], "free": s["free"], "count": s["count2"]}
    lay = Q4Layout(H=s["H"], d=s["d"], group=s["group"])
    if s["kind"] == "store":
        ops.q4_write_paged(lay, s["cache"], s["slots"], s["k"], s["v"], skip_pad=True)
        ops.q4_read_paged(lay, s["cache"], s["slots"], s["k_out"], s["v_out"], skip_pad=True)
        return {"k": s["k_out"], "v": s["v_out"]}
    if s["kind"] == "decode":
        return ops.q4_decode_paged(lay, s["cache"], s["table"], s["seq"], s["q"], s["scale"], s["out"])
    return ops.q4_prefill_paged(lay, s["cache"], s["table"], s["seq"], s["q_start"], s["q_len"], s["q"], s["scale"], s["out"],
                                s["max_q"], s["max_seq"])


def run(state):
    if own:
        return _own_run(state)
    if state["kind"] == "store":
        return _plain_store(state)
    if state["kind"] == "plan":
        return _plain_plan(state)
    return _plain_attend(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "store":
        n, H, d = case["tokens"], case["H"], case["d"]
        e = 4 if case["dtype"] == "fp32" else 2
        packed = n * H * (d + 8 * (d // case["group"]))
        # written: the values in, the packed rows out; read back: the packed rows in, the values out
        return {"bytes": 2 * (2 * n * H * d * e + packed + 8 * n), "flops": 12 * n * H * d}
    seq, ql, gone = _lengths(case, 0)
    if case["kind"] == "plan":
        seq, ql = seq[~gone], ql[~gone]
        new = int((-(-seq // case["block"]) - -(-(seq - ql) // case["block"])).sum())
        return {"bytes": 16 * int(ql.sum()) + 8 * new + 12 * case["reqs"], "flops": 4 * int(ql.sum())}
    row = case["H"] * (case["d"] + 8 * (case["d"] // case["group"]))
    pairs = int((ql * seq - ql * (ql - 1) // 2).sum())
    return {"bytes": int(seq.sum()) * row + 4 * int(ql.sum()) * case["HQ"] * case["d"] + 4 * int((-(-seq // case["block"])).sum()),
            "flops": 4 * pairs * case["HQ"] * case["d"]}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_token_values(panel, off, d, g):
    """K and V values (float64 numpy [d]) of token `off` of a panel's bytes, written out by lane."""
    lane = np.arange(d)
    kbyte = off * (d // 2) + ((lane % 32) // 8) * (d // 8) + (lane // 32) * 4 + (lane % 8) // 2
    vbyte = 8 * d + (off // 2) * d + ((lane % 32) // 4) * (d // 8) + (lane // 32) * 4 + (off % 2) * 2 + (lane % 4) // 2
    ng = d // g
    out = []
    for byte, base in ((kbyte, 16 * d), (vbyte, 16 * d + 64 * ng)):
        c = ((panel[..., byte] >> (4 * (lane % 2))) & 15).astype(np.float64)
        at = base + off * 4 * ng
        sm = np.ascontiguousarray(panel[..., at:at + 4 * ng]).view(np.float16).astype(np.float64)
        out.append(sm[..., 2 * (lane // g) + 1] + sm[..., 2 * (lane // g)] * c)
    return out


def _exact_store(s):
    out = {}
    keep = (s["slots"].cpu().numpy() >= 0)[:, None, None]
    for name in ("k", "v"):
        x = s[name].double().cpu().numpy()
        xg = np.clip(x, -LIMIT, LIMIT).reshape(*x.shape[:2], -1, s["group"])
        lo, hi = xg.min(-1, keepdims=True), xg.max(-1, keepdims=True)
        m = lo.astype(np.float16).astype(np.float64)
        sc = ((hi - lo) / 15.0).astype(np.float16).astype(np.float64)
        code = np.clip(np.rint((xg - m) / np.where(sc > 0, sc, 1.0)), 0, 15) * (sc > 0)
        out[name] = torch.from_numpy(np.where(keep, (m + sc * code).reshape(x.shape), 0.0))
    return out


def _exact_attend(s):
    d, g, bs, H = s["d"], s["group"], s["block"], s["H"]
    G = s["HQ"] // H
    cache, table = s["cache"], s["table"].cpu().numpy()
    seq, ql, q0 = (s[k].cpu().numpy().astype(np.int64) for k in ("seq", "q_len", "q_start"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r in range(s["reqs"]):
        n, nq = int(seq[r]), int(ql[r])
        blocks = torch.as_tensor(table[r, :-(-n // bs)].astype(np.int64), device=DEV)
        q = s["q"][q0[r]:q0[r] + nq].double()
        for h in range(H):
            pan = cache[blocks, h].reshape(-1, cache.shape[-1]).cpu().numpy()
            kv = [_exact_token_values(pan, o, d, g) for o in range(16)]
            K, V = (torch.from_numpy(np.stack([kv[o][i] for o in range(16)], 1).reshape(-1, d)[:n]).to(DEV) for i in (0, 1))
            late = torch.arange(n, device=DEV) > (n - nq + torch.arange(nq, device=DEV))[:, None]
            for i in range(G):
                sc = q[:, h * G + i] @ K.T * s["scale"]
                sc.masked_fill_(late, float("-inf"))
                out[q0[r]:q0[r] + nq, h * G + i] = torch.softmax(sc, -1) @ V
    return out


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(s)
    if int(s["seq"].sum()) * case["H"] * case["d"] > 200_000_000:
        return None
    return _exact_attend(s)
