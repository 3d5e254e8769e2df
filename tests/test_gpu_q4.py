"""The 4-bit paged cache on the GPU, against the 64-bit oracle (`oracle/q4.py`), through `vllm_ttkv.ops`.

Stored bytes and values that are read back are exact: the format rounds each scale, minimum and code
once. Tolerances of the attention, per output element, with e = half a step of the output's type
(2^-9 bf16 next to 2^-12 fp16, relative) and R = the largest |V| that the row sees:
  e |o|                       the output's own rounding
  2^-12 R                     the weights, rounded to fp16 (each acts on a value at most R off centre)
  2^-12 R                     everything in fp32: exponentials (2^-21), sums, scores
  2 * 2^-11 * A * R           chunks only: K and V read as fp16 (2^-11 of an element at most), where A is
                              the row's largest scale * sum |q_i K_i|, 1 at least (V's own share)
"""
import numpy as np
import pytest
import torch

from oracle import q4 as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GEOMETRIES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


def _lay(H, d, g):
    from vllm_ttkv.q4 import Q4Layout
    return Q4Layout(H=H, d=d, group=g)


def _np(t):
    return t.double().cpu().numpy()


def _filled(lay, seqs, bs, seed, dtype=torch.float32, poison=True):
    """(cache, block table, K, V values [per request]): each request's tokens written through
    `q4_write_paged`. Slots of no token hold NaN where `poison`."""
    from vllm_ttkv import ops
    rng = np.random.default_rng(seed)
    nb = [-(-n // bs) for n in seqs]
    total = sum(nb) + 2
    perm = rng.permutation(total)
    table = np.full((len(seqs), max(nb + [1]) + 1), total - 1, np.int64)
    cache = lay.new_cache(total, bs)
    if poison:
        cache.view(torch.float16).fill_(float("nan"))
    slots, at = [], 0
    for r, n in enumerate(seqs):
        table[r, :nb[r]] = perm[at:at + nb[r]]
        at += nb[r]
        t = np.arange(n)
        slots.append(table[r, t // bs] * bs + t % bs)
    slots = np.concatenate(slots).astype(np.int64)
    k = torch.from_numpy(rng.standard_normal((len(slots), lay.H, lay.d))).to(dtype).cuda()
    k[:, :, :3] *= 6
    v = torch.from_numpy(rng.standard_normal((len(slots), lay.H, lay.d))).to(dtype).cuda()
    ops.q4_write_paged(lay, cache, torch.from_numpy(slots).cuda(), k, v)
    K, V, at = [], [], 0
    for n in seqs:
        K.append(O.values(*O.quantise(_np(k[at:at + n]), lay.group)))
        V.append(O.values(*O.quantise(_np(v[at:at + n]), lay.group)))
        at += n
    return cache, torch.from_numpy(table).int().cuda(), K, V


def _check_rows(out, q, K, V, scale, G, dtype, chunk):
    want = O.attend(q, K, V, scale, G)
    e = torch.finfo(dtype).eps / 2
    for h in range(q.shape[1]):
        R = np.abs(V[:, h // G]).max()
        tol = e * np.abs(want[:, h]) + 2 * 2.0 ** -12 * R
        if chunk:
            A = max(1.0, abs(scale) * (np.abs(q[:, h]) @ np.abs(K[:, h // G]).T).max())
            tol = tol + 2 * 2.0 ** -11 * A * R
        err = np.abs(out[:, h] - want[:, h])
        assert np.all(err <= tol), (h, float((err / tol).max()), float(err.max()))


# ------------------------------------------------------------------ write and read-back
@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_store_bytes_and_values(d, g, dtype):
    from vllm_ttkv import ops
    lay, bs, n = _lay(3, d, g), 32, 45
    rng = np.random.default_rng(d + g)
    cache = lay.new_cache(5, bs)
    slots = rng.permutation(5 * bs)[:n]
    x = rng.standard_normal((2, n, 3, d)) * 10.0 ** rng.uniform(-6, 4, (2, n, 3, 1))
    x[0, 1] = 0.0                                      # a constant group: scale 0
    x[0, 2] = -3.25
    x[1, 3] = np.round(x[1, 3] * 8) / 8                # many quotients on a border
    x[0, 4] = np.tile(np.arange(16) / 2, d // 16)      # exact ties between codes
    x[1, 5] = 1000.0 + 1e-3 * x[1, 5]                  # a minimum far above the scale
    x[0, 6, :, 3], x[0, 6, :, 9] = 1e6, -1e6           # beyond the limit (infinite in fp16)
    x[1, 7, :, 5] = np.nan
    x[1, 8, :, 6] = np.inf
    x[0, 9] = 1e-7 * rng.standard_normal((3, d))       # scales below fp16's smallest normal
    k, v = (torch.from_numpy(a).to(DT[dtype]).cuda() for a in x)
    ops.reset_status()
    ops.q4_write_paged(lay, cache, torch.from_numpy(slots).cuda(), k, v)
    ops.check_status()
    want = np.zeros(tuple(cache.shape), np.uint8)
    kq, vq = O.quantise(_np(k), g), O.quantise(_np(v), g)
    for i, s in enumerate(slots):
        for h in range(3):
            O.put(want, s, h, bs, [a[i, h] for a in kq], [a[i, h] for a in vq])
    got = cache.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    for odt in (torch.float32, torch.float16, torch.bfloat16):
        ko, vo = torch.full_like(k, 7.0, dtype=odt), torch.full_like(v, 7.0, dtype=odt)
        ops.q4_read_paged(lay, cache, torch.from_numpy(slots).cuda(), ko, vo)
        for o, (c, s, m) in ((ko, kq), (vo, vq)):
            # m + s c rounded to fp32 (s c is exact), then to the type
            ref = torch.from_numpy(O.values(c, s, m)).float().to(odt)
            assert torch.equal(o.cpu().nan_to_num(nan=-1e4), ref.nan_to_num(nan=-1e4))
    ops.check_status()


@pytest.mark.parametrize("case", ["strided", "odd base", "one token", "none"])
def test_store_strides(case):
    """Rows of any stride and base: slices of a fused projection, a base off 16 bytes."""
    from vllm_ttkv import ops
    lay, bs = _lay(2, 64, 32), 16
    n = {"one token": 1, "none": 0}.get(case, 19)
    gen = torch.Generator().manual_seed(5)
    if case == "odd base":
        flat = torch.randn(2 * n * 128 + 3, generator=gen).half().cuda()
        k, v = flat[1:1 + n * 128].view(n, 2, 64), flat[n * 128 + 3:].view(n, 2, 64)
    else:
        qkv = torch.randn(n, 8, 64, generator=gen).half().cuda()
        k, v = qkv[:, 4:6], qkv[:, 6:8]
    slots = torch.arange(3, 3 + n, device="cuda")
    a, b = lay.new_cache(3, bs), lay.new_cache(3, bs)
    ops.q4_write_paged(lay, a, slots, k, v)
    ops.q4_write_paged(lay, b, slots, k.contiguous().clone(), v.contiguous().clone())
    assert torch.equal(a, b)
    wide = torch.full((n, 8, 64), 9.0, device="cuda", dtype=torch.float16)
    ko, vo = torch.zeros(n, 2, 64, device="cuda").half(), torch.zeros(n, 2, 64, device="cuda").half()
    ops.q4_read_paged(lay, a, slots, ko, vo)
    ops.q4_read_paged(lay, a, slots, wide[:, 4:6], wide[:, 6:8])
    assert torch.equal(wide[:, 4:6], ko) and torch.equal(wide[:, 6:8], vo)
    assert bool((wide[:, :4] == 9).all())
    ops.check_status()


@pytest.mark.parametrize("kt,vt", [("bf16", "fp32"), ("fp32", "fp16"), ("fp16", "bf16")])
def test_store_of_two_types(kt, vt):
    from vllm_ttkv import ops
    lay, bs = _lay(2, 128, 32), 16
    gen = torch.Generator().manual_seed(5)
    k, v = torch.randn(40, 2, 128, generator=gen).to(DT[kt]).cuda(), torch.randn(40, 2, 128, generator=gen).to(DT[vt]).cuda()
    slots = torch.arange(5, 45, device="cuda")
    a, b = lay.new_cache(3, bs), lay.new_cache(3, bs)
    ops.q4_write_paged(lay, a, slots, k, v)
    ops.q4_write_paged(lay, b, slots, k.float(), v.float())
    assert torch.equal(a, b)
    ko, vo, kf, vf = torch.empty_like(k), torch.empty_like(v), torch.empty_like(k).float(), torch.empty_like(v).float()
    ops.q4_read_paged(lay, a, slots, ko, vo)
    ops.q4_read_paged(lay, a, slots, kf, vf)
    assert torch.equal(ko, kf.to(DT[kt])) and torch.equal(vo, vf.to(DT[vt]))


def test_store_skips_and_refuses_slots():
    from vllm_ttkv import ops
    lay, bs = _lay(1, 128, 64), 16
    cache = lay.new_cache(2, bs)
    k = torch.randn(4, 1, 128, device="cuda")
    slots = torch.tensor([3, -1, 32, 5], device="cuda")
    ops.reset_status()
    ops.q4_write_paged(lay, cache, slots[[0, 1, 3]].contiguous(), k, k, skip_pad=True)
    ops.check_status()
    ko = torch.full((4, 1, 128), 3.0, device="cuda")
    vo = ko.clone()
    ops.q4_read_paged(lay, cache, slots, ko, vo, skip_pad=True)
    with pytest.raises(IndexError):                    # slot 32 is outside the 2 blocks
        ops.check_status()
    assert bool((ko[1:3] == 3).all()) and bool((vo[1:3] == 3).all()) and not bool((ko[0] == 3).any())
    before = cache.clone()
    ops.q4_write_paged(lay, cache, slots[1:3].contiguous(), k, k)
    with pytest.raises(IndexError):
        ops.check_status()
    assert torch.equal(cache, before)


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("H,HQ,dtype,bs", [(1, 1, "fp16", 16), (2, 6, "bf16", 16), (2, 16, "fp16", 64), (1, 13, "bf16", 32),
                                           (3, 60, "fp16", 16)])
def test_decode(d, g, H, HQ, dtype, bs):
    from vllm_ttkv import ops
    lay = _lay(H, d, g)
    seqs = [0, 1, 15, 16, 17, 63, 64, 65, 200, 0, 1031]
    cache, table, K, V = _filled(lay, seqs, bs, seed=HQ + d)
    q = torch.randn(len(seqs), HQ, d, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.full_like(q, 5.0)
    ops.reset_status()
    ops.q4_decode_paged(lay, cache, table, torch.tensor(seqs, dtype=torch.int32, device="cuda"), q, d ** -0.5, out)
    ops.check_status()
    for r, n in enumerate(seqs):
        if n == 0:
            assert not bool(out[r].any())
        else:
            _check_rows(_np(out[r:r + 1]), _np(q[r:r + 1]), K[r], V[r], d ** -0.5, HQ // H, DT[dtype], False)


@pytest.mark.parametrize("B,n,H,HQ", [(1, 9000, 1, 4), (300, 40, 2, 2), (5, 2500, 2, 24), (530, 3, 1, 1)])
def test_decode_splits(B, n, H, HQ):
    """Few long requests (parts of many CTAs joined) and many short ones (many requests per warp)."""
    from vllm_ttkv import ops
    lay = _lay(H, 64, 64)
    rng = np.random.default_rng(B)
    seqs = [int(x) for x in rng.integers(max(1, n // 2), n + 1, B)]
    cache, table, K, V = _filled(lay, seqs, 16, seed=B)
    q = torch.randn(B, HQ, 64, generator=torch.Generator().manual_seed(B)).half().cuda()
    out = torch.empty_like(q)
    ops.q4_decode_paged(lay, cache, table, torch.tensor(seqs, dtype=torch.int32, device="cuda"), q, 0.2, out)
    ops.check_status()
    for r in range(B):
        _check_rows(_np(out[r:r + 1]), _np(q[r:r + 1]), K[r], V[r], 0.2, HQ // H, torch.float16, False)


@pytest.mark.parametrize("kscale,vscale,qscale", [(1, 1e-4, 1), (1, 3e3, 1), (30, 1, 1e-3), (1e-3, 1, 300), (0, 1, 1), (1, 0, 1)])
def test_decode_ranges(kscale, vscale, qscale):
    """Values far from 1: weights are scaled with the V scales that they meet, queries by their size.
    Constant values (scale 0) are read from the minimum alone."""
    from vllm_ttkv import ops
    lay, n = _lay(1, 128, 128), 333
    rng = np.random.default_rng(9)
    k = torch.from_numpy(rng.standard_normal((n, 1, 128)) * kscale).float().cuda()
    v = torch.from_numpy(rng.standard_normal((n, 1, 128)) * vscale * 10.0 ** rng.uniform(-2, 0, (n, 1, 1))).float().cuda()
    if vscale == 0:
        v += torch.from_numpy(rng.standard_normal((n, 1, 1))).float().cuda()
    cache = lay.new_cache(30, 16)
    table = torch.randperm(30, generator=torch.Generator().manual_seed(1)).int()[None].cuda()
    t = torch.arange(n, device="cuda")
    ops.q4_write_paged(lay, cache, table[0].long()[t // 16] * 16 + t % 16, k, v)
    q = (torch.from_numpy(rng.standard_normal((1, 5, 128))) * qscale).half().cuda()
    out = torch.empty_like(q)
    ops.q4_decode_paged(lay, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), q, 0.1, out)
    K, V = (O.values(*O.quantise(_np(x), 128)) for x in (k, v))
    _check_rows(_np(out), _np(q), K, V, 0.1, 5, torch.float16, False)


def test_decode_reads_nan_of_a_token_and_no_other():
    """A NaN that a request has stored reaches its outputs; one in the slots of nobody does not (every
    store of these tests is poisoned), nor one behind the request's end in its own last block."""
    from vllm_ttkv import ops
    lay = _lay(1, 64, 32)
    seqs = [20, 20]
    cache, table, K, V = _filled(lay, seqs, 16, seed=4)
    bad = torch.full((1, 1, 64), float("nan"), device="cuda")
    slot = table[1, 0].long()[None] * 16 + 7
    ops.q4_write_paged(lay, cache, slot, torch.zeros_like(bad), bad)
    q = torch.randn(2, 2, 64, device="cuda").half()
    out = torch.empty_like(q)
    ops.q4_decode_paged(lay, cache, table, torch.tensor(seqs, dtype=torch.int32, device="cuda"), q, 0.1, out)
    assert bool(out[1].isnan().all())
    _check_rows(_np(out[:1]), _np(q[:1]), K[0], V[0], 0.1, 2, torch.float16, False)


def test_decode_refusals_on_the_device():
    from vllm_ttkv import ops
    lay = _lay(2, 64, 64)
    seqs = [40, 40, 40]
    cache, table, K, V = _filled(lay, seqs, 16, seed=4)
    q = torch.randn(3, 4, 64, device="cuda").half()
    sl = torch.tensor([40, 40, 40], dtype=torch.int32, device="cuda")
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t2 = table.clone()
        t2[1, 1] = bad
        out = torch.full_like(q, 5.0)
        ops.reset_status()
        ops.q4_decode_paged(lay, cache, t2, sl, q, 0.1, out)
        with pytest.raises(IndexError):
            ops.check_status()
        assert bool(out[1].isnan().all())
        for r in (0, 2):
            _check_rows(_np(out[r:r + 1]), _np(q[r:r + 1]), K[r], V[r], 0.1, 2, torch.float16, False)
    sl[1] = 16 * table.shape[1] + 1                     # more tokens than the row has blocks
    out = torch.full_like(q, 5.0)
    ops.q4_decode_paged(lay, cache, table, sl, q, 0.1, out)
    with pytest.raises(RuntimeError):
        ops.check_status()
    assert bool((out[1] == 5).all()) and not bool((out[0] == 5).any())


def test_decode_strides_and_offsets():
    """Queries that are slices of a fused projection, a base off 16 bytes, an output with gaps."""
    from vllm_ttkv import ops
    lay, seqs = _lay(2, 64, 64), [70, 5]
    cache, table, K, V = _filled(lay, seqs, 16, seed=8)
    sl = torch.tensor(seqs, dtype=torch.int32, device="cuda")
    qkv = torch.randn(2, 10, 64, device="cuda").to(torch.bfloat16)
    big = torch.full((2 * 10 * 64 + 1,), 9.0, device="cuda", dtype=torch.bfloat16)
    wide = big[1:].view(2, 10, 64)
    ops.q4_decode_paged(lay, cache, table, sl, qkv[:, :6], 0.1, wide[:, 2:8])
    shifted = torch.empty(2 * 6 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    shifted[1:] = qkv[:, :6].reshape(-1)
    out = torch.empty(2, 6, 64, device="cuda", dtype=torch.bfloat16)
    ops.q4_decode_paged(lay, cache, table, sl, shifted[1:].view(2, 6, 64), 0.1, out)
    assert torch.equal(out, wide[:, 2:8])
    assert bool((wide[:, :2] == 9).all()) and bool((wide[:, 8:] == 9).all())
    for r in range(2):
        _check_rows(_np(out[r:r + 1]), _np(qkv[r:r + 1, :6]), K[r], V[r], 0.1, 3, torch.bfloat16, False)


def test_decode_captured_and_on_two_streams():
    """A captured call replays other lengths; two graphs and eager calls on other streams run at once
    without sharing scratch."""
    from vllm_ttkv import ops
    lay, seqs = _lay(1, 128, 64), [700, 3000, 65]
    cache, table, K, V = _filled(lay, seqs, 16, seed=2)
    q = torch.randn(3, 8, 128, device="cuda").half()
    ops.status_word()
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seqs, seqs)]
    outs = [torch.empty_like(q) for _ in range(3)]
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.q4_decode_paged(lay, cache, table, lens[i], q, 0.1, outs[i])
        graphs.append(g)
    lens[0].copy_(torch.tensor([1, 2000, 0], dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            ops.q4_decode_paged(lay, cache, table, lens[1], q, 0.1, outs[2])
    torch.cuda.synchronize()
    assert torch.equal(outs[1], outs[2]) and not bool(outs[0][2].any())
    for o, ns in ((outs[0], [1, 2000]), (outs[1], seqs)):
        for r, n in enumerate(ns):
            _check_rows(_np(o[r:r + 1]), _np(q[r:r + 1]), K[r][:n], V[r][:n], 0.1, 8, torch.float16, False)


# ------------------------------------------------------------------ chunks
def _prefill(lay, cache, table, seqs, qls, q, scale, out, gap=0, max_q=None, max_seq=None):
    from vllm_ttkv import ops
    starts, at = [], 0
    for n in qls:
        starts.append(at)
        at += n + gap
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.q4_prefill_paged(lay, cache, table, i32(seqs), i32(starts), i32(qls), q, scale, out,
                         max(qls) if max_q is None else max_q, max(seqs) if max_seq is None else max_seq)
    return starts


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("H,HQ,dtype,bs", [(1, 1, "fp16", 16), (2, 6, "bf16", 16), (1, 13, "fp16", 64)])
@pytest.mark.parametrize("qls", [(1, 4, 0, 2), (1, 127, 128, 129), (300, 0, 33, 65)])
def test_prefill(d, g, H, HQ, dtype, bs, qls):
    from vllm_ttkv import ops
    lay = _lay(H, d, g)
    seqs = [n + extra if n else 0 for n, extra in zip(qls, (0, 130, 5, 333))]
    cache, table, K, V = _filled(lay, seqs, bs, seed=HQ + d)
    gap = 2
    q = torch.randn(sum(qls) + gap * len(qls), HQ, d, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.full_like(q, 5.0)
    ops.reset_status()
    starts = _prefill(lay, cache, table, seqs, qls, q, d ** -0.5, out, gap)
    ops.check_status()
    for r, (a, n) in enumerate(zip(starts, qls)):
        if n:
            _check_rows(_np(out[a:a + n]), _np(q[a:a + n]), K[r], V[r], d ** -0.5, HQ // H, DT[dtype], True)
        assert bool((out[a + n:a + n + gap] == 5).all())         # rows of no request


@pytest.mark.parametrize("H,HQ,ql,n", [(1, 2, 200, 5000), (2, 8, 33, 3001), (1, 16, 9, 9000)])
def test_prefill_splits(H, HQ, ql, n):
    """Few rows over many tokens: parts along the tokens joined."""
    from vllm_ttkv import ops
    lay = _lay(H, 128, 128)
    cache, table, K, V = _filled(lay, [n], 16, seed=ql)
    q = torch.randn(ql, HQ, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, 0.08, out)
    ops.check_status()
    _check_rows(_np(out), _np(q), K[0], V[0], 0.08, HQ // H, torch.float16, True)


@pytest.mark.parametrize("R,H,ql", [(40, 1, 4), (40, 1, 6), (40, 1, 7), (40, 1, 8), (40, 1, 9), (3, 2, 12), (3, 2, 16),
                                    (3, 2, 17), (17, 2, 12)])
def test_prefill_streamed_or_not(R, H, ql):
    """Row counts, batches and bounds on both sides of the choice between the two kernels."""
    from vllm_ttkv import ops
    lay = _lay(H, 128, 64) if R == 3 else _lay(H, 64, 64)
    rng = np.random.default_rng(ql)
    seqs = [ql + int(x) for x in rng.integers(0, 300, R)]
    cache, table, K, V = _filled(lay, seqs, 16, seed=R)
    q = torch.randn(R * ql, 4 * H, lay.d, generator=torch.Generator().manual_seed(3)).half().cuda()
    for bound in (max(seqs), 1535, 1536, 100000):
        out = torch.empty_like(q)
        starts = _prefill(lay, cache, table, seqs, [ql] * R, q, 0.125, out, max_seq=bound)
        ops.check_status()
        for r, a in enumerate(starts):
            _check_rows(_np(out[a:a + ql]), _np(q[a:a + ql]), K[r], V[r], 0.125, 4, torch.float16, True)


@pytest.mark.parametrize("d,g", GEOMETRIES)
def test_prefill_many_tiles(d, g):
    """Some 40 stored tiles a CTA: every place of its ring of panels is filled again and again. The requests
    share one sequence's blocks."""
    from vllm_ttkv import ops
    lay, R, ql, n, G = _lay(1, d, g), 64, 64, 6000, 8
    cache, table, K, V = _filled(lay, [n], 16, seed=d + g)
    q = torch.randn(R * ql, G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table.expand(R, -1), [n - 3 * r for r in range(R)], [ql] * R, q, 0.05, out)
    ops.check_status()
    for r in (0, 23, 47, 63):
        a, m = starts[r], n - 3 * r
        _check_rows(_np(out[a:a + ql]), _np(q[a:a + ql]), K[0][:m], V[0][:m], 0.05, G, torch.float16, True)
    again = torch.empty_like(q)
    _prefill(lay, cache, table.expand(R, -1), [n - 3 * r for r in range(R)], [ql] * R, q, 0.05, again)
    assert torch.equal(out, again)


def test_prefill_a_nan_reaches_the_queries_that_see_it():
    from vllm_ttkv import ops
    lay = _lay(1, 64, 32)
    for ql, n in ((6, 100), (150, 300)):
        cache, table, K, V = _filled(lay, [n], 16, seed=4)
        at = n - 3                                       # seen by the last three queries only
        bad = torch.full((1, 1, 64), float("nan"), device="cuda")
        slot = table[0, at // 16].long()[None] * 16 + at % 16
        ops.q4_write_paged(lay, cache, slot, bad, bad)
        q = torch.randn(ql, 2, 64, device="cuda").half()
        out = torch.empty_like(q)
        _prefill(lay, cache, table, [n], [ql], q, 0.1, out)
        assert bool(out[-3:].isnan().all())
        _check_rows(_np(out[:-3]), _np(q[:-3]), K[0][:at], V[0][:at], 0.1, 2, torch.float16, True)


def test_prefill_refusals_on_the_device():
    from vllm_ttkv import ops
    lay = _lay(1, 64, 64)
    for ql in (4, 140):
        seqs, qls = [ql + 20, ql + 50, ql], [ql, ql, ql]
        cache, table, K, V = _filled(lay, seqs, 16, seed=4)
        q = torch.randn(3 * ql, 2, 64, device="cuda").half()
        for seqs2, qls2, kw, exc in (([ql + 20, ql - 1, ql], qls, {}, RuntimeError),
                                     (seqs, qls, dict(max_seq=ql + 20), RuntimeError),
                                     (seqs, [ql - 1, ql, ql - 1], dict(max_q=ql - 1), RuntimeError),
                                     ([ql + 20, 16 * table.shape[1] + 1, ql], qls, dict(max_seq=10 ** 6), RuntimeError)):
            out = torch.full_like(q, 5.0)
            ops.reset_status()
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            ops.q4_prefill_paged(lay, cache, table, i32(seqs2), i32([0, ql, 2 * ql]), i32(qls2), q, 0.1, out,
                                 kw.get("max_q", ql), kw.get("max_seq", max(seqs2)))
            with pytest.raises(exc):
                ops.check_status()
            assert bool((out[ql:2 * ql] == 5).all())
            for r in (0, 2):
                a, n = r * ql, qls2[r]
                K2, V2 = K[r][:seqs2[r]], V[r][:seqs2[r]]
                _check_rows(_np(out[a:a + n]), _np(q[a:a + n]), K2, V2, 0.1, 2, torch.float16, True)
        t2 = table.clone()
        t2[1, 1] = -1
        out = torch.full_like(q, 5.0)
        ops.reset_status()
        _prefill(lay, cache, t2, seqs, qls, q, 0.1, out)
        with pytest.raises(IndexError):
            ops.check_status()
        assert bool(out[ql:2 * ql][-1].isnan().all())
        _check_rows(_np(out[:ql]), _np(q[:ql]), K[0], V[0], 0.1, 2, torch.float16, True)
        # query rows outside the tensor
        out = torch.full_like(q, 5.0)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        ops.q4_prefill_paged(lay, cache, table, i32(seqs), i32([0, 2 * ql + 1, -1]), i32(qls), q, 0.1, out, ql, max(seqs))
        with pytest.raises(RuntimeError):
            ops.check_status()
        assert bool((out[ql:] == 5).all())


def test_prefill_bounds_of_nothing():
    """No tokens allowed: every request is refused. No queries allowed: nothing is done."""
    from vllm_ttkv import ops
    lay = _lay(1, 64, 64)
    cache, table, K, V = _filled(lay, [1, 1], 16, seed=4)
    q = torch.randn(2, 2, 64, device="cuda").half()
    out = torch.full_like(q, 5.0)
    ops.reset_status()
    _prefill(lay, cache, table, [1, 1], [1, 1], q, 0.1, out, max_seq=0)
    with pytest.raises(RuntimeError):
        ops.check_status()
    _prefill(lay, cache, table, [1, 1], [1, 1], q, 0.1, out, max_q=0)
    ops.check_status()
    assert bool((out == 5).all())
    _prefill(lay, cache, table, [1, 1], [1, 1], q, 0.1, out, max_seq=1)
    ops.check_status()
    for r in range(2):
        _check_rows(_np(out[r:r + 1]), _np(q[r:r + 1]), K[r], V[r], 0.1, 2, torch.float16, True)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError):
            _prefill(lay, cache, table, [1, 1], [1, 1], q, scale, out)


def test_prefill_captured():
    from vllm_ttkv import ops
    lay = _lay(1, 128, 128)
    cache, table, K, V = _filled(lay, [900, 400], 16, seed=2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    seq, qs, ql = i32([900, 400]), i32([0, 160]), i32([160, 70])
    q = torch.randn(230, 2, 128, device="cuda").half()
    out = torch.full_like(q, 5.0)
    ops.status_word()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.q4_prefill_paged(lay, cache, table, seq, qs, ql, q, 0.1, out, 160, 1000)
    for seqs, qls in (([900, 400], [160, 70]), ([130, 399], [130, 1]), ([640, 0], [5, 0])):
        seq.copy_(i32(seqs))
        ql.copy_(i32(qls))
        out.fill_(5.0)
        g.replay()
        ops.check_status()
        for r, a in ((0, 0), (1, 160)):
            n = qls[r]
            if n:
                _check_rows(_np(out[a:a + n]), _np(q[a:a + n]), K[r][:seqs[r]], V[r][:seqs[r]], 0.1, 2, torch.float16, True)
            assert bool((out[a + n:(160, 230)[r]] == 5).all())


# ------------------------------------------------------------------ together
def test_serving_run():
    """A few requests served as an engine would: plan the step's blocks, write its tokens, attend, release;
    every output against dense attention over the values that the cache holds."""
    from vllm_ttkv import ops
    lay, bs, HQ, dt = _lay(2, 64, 32), 16, 6, torch.float16
    n_blocks, width, T = 40, 12, 64
    rng = np.random.default_rng(0)
    dev = "cuda"
    cache = lay.new_cache(n_blocks, bs)
    cache.view(torch.float16).fill_(float("nan"))
    free = torch.arange(n_blocks, dtype=torch.int32, device=dev)
    count = torch.tensor([n_blocks], dtype=torch.int32, device=dev)
    table = torch.full((3, width), -1, dtype=torch.int32, device=dev)
    slots, pos = torch.zeros(T, dtype=torch.int64, device=dev), torch.zeros(T, dtype=torch.int64, device=dev)
    lens, store = [0, 0, 0], [[[], []] for _ in range(3)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ops.reset_status()
    for step, qls in enumerate([(40, 3, 0), (17, 1, 21), (1, 1, 1), (1, 1, 1), (1, 0, 50), (1, 33, 1), (1, 1, 1)]):
        if step == 5:                                    # request 0 ends; its row serves a new one
            ops.release_blocks(table, i32([lens[0], 0, 0]), free, count, bs)
            lens[0], store[0] = 0, [[], []]
        lens = [a + b for a, b in zip(lens, qls)]
        qsl = np.concatenate([[0], np.cumsum(qls)])
        ops.plan_step(table, i32(lens), i32(qsl), free, count, bs, slots, positions=pos)
        k, v = (torch.from_numpy(rng.standard_normal((T, 2, 64))).to(dt).to(dev) for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((T, HQ, 64))).to(dt).to(dev)
        ops.q4_write_paged(lay, cache, slots, k, v, skip_pad=True)
        out = torch.full_like(q, 5.0)
        if max(qls) == 1 and min(qls) == 1:
            ops.q4_decode_paged(lay, cache, table, i32(lens), q[:3], 0.125, out)
        else:
            ops.q4_prefill_paged(lay, cache, table, i32(lens), i32(qsl[:-1]), i32(qls), q, 0.125, out, max(qls), max(lens))
        ops.check_status()
        for r in range(3):
            a, b = qsl[r], qsl[r + 1]
            for x, s in ((k, store[r][0]), (v, store[r][1])):
                s.append(O.values(*O.quantise(_np(x[a:b]), 32)))
            assert pos[a:b].tolist() == list(range(lens[r] - qls[r], lens[r]))
            if b > a:
                K, V = (np.concatenate(s) for s in store[r])
                _check_rows(_np(out[a:b]), _np(q[a:b]), K, V, 0.125, 3, dt, True)
        held = sum(-(-n // bs) for n in lens)
        assert int(count) == n_blocks - held


# ------------------------------------------------------------------ what the documentation allows besides
@pytest.mark.parametrize("bs", [48, 80, 2048])
@pytest.mark.parametrize("ql", [1, 3, 150])
def test_block_sizes(bs, ql):
    """Units of 64 tokens and tiles of 128 that begin and end inside blocks."""
    lay, seqs = _lay(2, 64, 32), [ql, 47 + ql, 1000 + ql]
    cache, table, K, V = _filled(lay, seqs, bs, seed=bs)
    q = torch.randn(3 * ql, 4, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table, seqs, [ql] * 3, q, 0.125, out)
    for r, a in enumerate(starts):
        _check_rows(_np(out[a:a + ql]), _np(q[a:a + ql]), K[r], V[r], 0.125, 2, torch.float16, True)


@pytest.mark.parametrize("ql", [1, 100])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales_of_any_sign(ql, scale):
    lay, n = _lay(1, 128, 64), 400
    cache, table, K, V = _filled(lay, [n], 16, seed=1)
    q = torch.randn(ql, 3, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, scale, out)
    _check_rows(_np(out), _np(q), K[0], V[0], scale, 3, torch.float16, True)


@pytest.mark.parametrize("ql", [2, 140])
def test_a_query_of_no_number_spoils_its_own_row_alone(ql):
    lay, n = _lay(1, 64, 32), 500
    cache, table, K, V = _filled(lay, [n], 16, seed=1)
    q = torch.randn(ql, 4, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    q[1, 2, 5], q[ql - 1, 0, 9] = float("nan"), float("inf")
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, 0.125, out)
    bad = torch.zeros(ql, 4, dtype=torch.bool)
    bad[1, 2] = bad[ql - 1, 0] = True
    assert bool(out[bad.cuda()].isnan().all())
    want = q.clone()
    want[bad.cuda()] = 0.0
    out[bad.cuda()] = torch.from_numpy(O.attend(_np(want), K[0], V[0], 0.125, 4))[bad].half().cuda()
    _check_rows(_np(out), _np(want), K[0], V[0], 0.125, 4, torch.float16, True)


def test_prefill_strides_and_offsets():
    """Chunks whose queries are slices of a fused projection or lie off 16 bytes, outputs with gaps."""
    lay, seqs, qls = _lay(2, 64, 64), [200, 77], [130, 60]
    cache, table, K, V = _filled(lay, seqs, 16, seed=8)
    T = sum(qls)
    qkv = torch.randn(T, 10, 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    big = torch.full((T * 10 * 64 + 1,), 9.0, device="cuda", dtype=torch.bfloat16)
    wide = big[1:].view(T, 10, 64)
    _prefill(lay, cache, table, seqs, qls, qkv[:, :6], 0.1, wide[:, 2:8])
    shifted = torch.empty(T * 6 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    shifted[1:] = qkv[:, :6].reshape(-1)
    out = torch.empty(T, 6, 64, device="cuda", dtype=torch.bfloat16)
    _prefill(lay, cache, table, seqs, qls, shifted[1:].view(T, 6, 64), 0.1, out)
    assert torch.equal(out, wide[:, 2:8])
    assert bool((wide[:, :2] == 9).all()) and bool((wide[:, 8:] == 9).all())
    for r, (a, n) in enumerate(((0, 130), (130, 60))):
        _check_rows(_np(out[a:a + n]), _np(qkv[a:a + n, :6]), K[r], V[r], 0.1, 3, torch.bfloat16, True)


def test_offsets_behind_32_bits():
    """A cache beyond 2^32 bytes, and rows of k, v, q and out more than 2^31 elements apart."""
    from vllm_ttkv import ops
    lay, bs = _lay(2, 128, 128), 16
    n_blocks = 2 ** 32 // (2 * lay.panel_bytes) + 50
    cache = torch.empty(lay.cache_shape(n_blocks, bs), dtype=torch.uint8, device="cuda")
    stride = 2 ** 30 + 64
    flat = torch.empty(3 * stride, dtype=torch.float16, device="cuda")

    def apart(n, heads, at):
        return torch.as_strided(flat, (n, heads, 128), (stride, 128, 1), at)

    gen = torch.Generator().manual_seed(0)
    blocks = [n_blocks - 1, 3, n_blocks - 30, n_blocks - 7, n_blocks // 2, 0, n_blocks - 2]
    n = 16 * len(blocks) - 5
    table = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    t = torch.arange(n, device="cuda")
    slots = table[0].long()[t // bs] * bs + t % bs
    k, v = (torch.randn(n, 2, 128, generator=gen).half().cuda() for _ in range(2))
    ops.reset_status()
    ops.q4_write_paged(lay, cache, slots[:-3], k[:-3], v[:-3])
    kf, vf = apart(3, 2, 0), apart(3, 2, 4096)
    kf.copy_(k[-3:])
    vf.copy_(v[-3:])
    ops.q4_write_paged(lay, cache, slots[-3:], kf, vf)
    ko, vo = apart(3, 2, 8192), apart(3, 2, 12288)
    ops.q4_read_paged(lay, cache, slots[-3:], ko, vo)
    K, V = (O.values(*O.quantise(_np(x), 128)) for x in (k, v))
    assert torch.equal(ko.cpu(), torch.from_numpy(K[-3:]).half()) and torch.equal(vo.cpu(), torch.from_numpy(V[-3:]).half())
    for heads, ql in ((4, 1), (4, 3), (32, 3)):          # streamed, and a chunk
        q, out = apart(ql, heads, 16384), apart(ql, heads, 32768)
        q.copy_(torch.randn(ql, heads, 128, generator=gen).half())
        if ql == 1:
            ops.q4_decode_paged(lay, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), q, 0.08, out)
        else:
            _prefill(lay, cache, table, [n], [ql], q, 0.08, out)
        ops.check_status()
        _check_rows(_np(out), _np(q), K, V, 0.08, heads // 2, torch.float16, True)


def test_many_heads_a_group_and_many_requests_of_a_chunk():
    from vllm_ttkv import ops
    lay = _lay(1, 64, 64)
    cache, table, K, V = _filled(lay, [300, 70], 16, seed=6)
    q = torch.randn(2, 71, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    ops.q4_decode_paged(lay, cache, table, torch.tensor([300, 70], dtype=torch.int32, device="cuda"), q, 0.1, out)
    for r in range(2):
        _check_rows(_np(out[r:r + 1]), _np(q[r:r + 1]), K[r], V[r], 0.1, 71, torch.float16, False)
    rng = np.random.default_rng(1)
    qls = [int(x) for x in rng.integers(0, 4, 400)]
    qls[200] = 90
    seqs = [n + int(x) if n else 0 for n, x in zip(qls, rng.integers(0, 60, 400))]
    cache, table, K, V = _filled(lay, seqs, 16, seed=7)
    q = torch.randn(sum(qls), 2, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table, seqs, qls, q, 0.1, out)
    ops.check_status()
    for r, (a, n) in enumerate(zip(starts, qls)):
        if n:
            _check_rows(_np(out[a:a + n]), _np(q[a:a + n]), K[r], V[r], 0.1, 2, torch.float16, True)


def test_prefill_in_two_graphs_at_once():
    """Two captured chunk calls and an eager one, replayed at once on three streams: no shared scratch, and
    each answer the same bits every time."""
    from vllm_ttkv import ops
    lay, seqs, qls = _lay(1, 128, 128), [2500, 700], [100, 64]
    cache, table, K, V = _filled(lay, seqs, 16, seed=2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    seq, qs, ql = i32(seqs), i32([0, 100]), i32(qls)
    qq = [torch.randn(164, 4, 128, generator=torch.Generator().manual_seed(i)).half().cuda() for i in range(3)]
    outs = [torch.empty_like(x) for x in qq]
    want = [torch.empty_like(x) for x in qq]
    ops.status_word()

    def call(i, out):
        ops.q4_prefill_paged(lay, cache, table, seq, qs, ql, qq[i], 0.1, out[i], 100, 2500)

    for i in range(3):
        call(i, want)
        for r, (a, n) in enumerate(((0, 100), (100, 64))):
            _check_rows(_np(want[i][a:a + n]), _np(qq[i][a:a + n]), K[r], V[r], 0.1, 4, torch.float16, True)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(i, outs)
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for i in range(3):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay() if i < 2 else call(2, outs)
    torch.cuda.synchronize()
    ops.check_status()
    for i in range(3):
        assert torch.equal(outs[i], want[i])


# ------------------------------------------------------------------ refusals before a launch
def test_the_binding_refuses_other_types():
    from vllm_ttkv import ops
    lay = _lay(1, 64, 64)
    cache = lay.new_cache(2, 16)
    kv, sl = torch.zeros(3, 1, 64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    i32 = torch.zeros(3, dtype=torch.int32, device="cuda")
    bt, q = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), kv.half()
    for call in (lambda: ops.q4_write_paged(lay, None, sl, kv, kv), lambda: ops.q4_write_paged(lay, cache, [0, 1, 2], kv, kv),
                 lambda: ops.q4_write_paged(lay, cache, sl, kv.cpu().numpy(), kv), lambda: ops.q4_write_paged(lay, cache, sl, kv, 3),
                 lambda: ops.q4_write_paged(lay, cache, sl, kv, kv, status=7),
                 lambda: ops.q4_decode_paged(lay, cache, bt, i32, q, "a", q), lambda: ops.q4_decode_paged(lay, cache, bt, i32, q, None, q),
                 lambda: ops.q4_prefill_paged(lay, cache, bt, i32, i32, i32, q, 1.0, q, 1.5, 1),
                 lambda: ops.q4_prefill_paged(lay, cache, bt, i32, i32, i32, q, 1.0, q, 1, None),
                 lambda: ops.plan_step(bt, i32, i32, i32, i32[:1], "16", sl), lambda: ops.release_blocks(bt, i32, None, i32[:1], 16)):
        with pytest.raises((TypeError, ValueError, AttributeError)):
            call()
    for call in (lambda: ops.q4_prefill_paged(lay, cache, bt, i32, i32, i32, q, 1.0, q, 2 ** 40, 1),
                 lambda: ops.q4_prefill_paged(lay, cache, bt, i32, i32, i32, q, 1.0, q, 2 ** 70, 1)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


def test_ops_refuse_what_does_not_fit():
    from vllm_ttkv import ops
    lay = _lay(2, 64, 32)
    cache = lay.new_cache(4, 16)
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    kv, sl = z(3, 2, 64), z(3, dt=i64)
    for args in ((cache[:, :1], sl, kv, kv), (cache, sl.int(), kv, kv), (cache, z(6, dt=i64)[::2], kv, kv), (cache, sl, kv[:2], kv),
                 (cache, sl, z(3, 1, 64), kv), (cache, sl, kv, z(3, 2, 32)), (cache, sl, kv.double(), kv),
                 (cache, sl, z(3, 64, 2).transpose(1, 2), kv), (cache, sl, kv.cpu(), kv), (cache, sl.cpu(), kv, kv),
                 (cache, sl, kv[:1].expand(3, 2, 64), kv)):
        for fn in (ops.q4_write_paged, ops.q4_read_paged):
            with pytest.raises((TypeError, ValueError)):
                fn(lay, *args)
    bt, sq, q = z(3, 4, dt=i32), z(3, dt=i32), z(3, 4, 64)
    for args in ((cache.int(), bt, sq, q, 1.0, q), (cache, bt.long(), sq, q, 1.0, q), (cache, bt[:2], sq, q, 1.0, q),
                 (cache, bt.t(), sq, q[:4], 1.0, q), (cache, bt, sq[:2], q, 1.0, q), (cache, bt, sq.long(), q, 1.0, q),
                 (cache, bt, sq, q.float(), 1.0, q.float()), (cache, bt, sq, q, 1.0, q.bfloat16()), (cache, bt, sq, q, 1.0, q[:2]),
                 (cache, bt, sq, q[:, :3], 1.0, q[:, :3]), (cache, bt, sq, q, 1.0, q[:, :2]), (cache, bt, sq.cpu(), q, 1.0, q)):
        with pytest.raises((TypeError, ValueError)):
            ops.q4_decode_paged(lay, *args)
    for args in ((cache, bt, sq, sq.long(), sq, q, 1.0, q, 1, 1), (cache, bt, sq, sq[:2], sq, q, 1.0, q, 1, 1),
                 (cache, bt, sq, sq, sq, q, 1.0, q, -1, 1), (cache, bt, sq, sq, sq, q, 1.0, q[:2], 1, 1)):
        with pytest.raises((TypeError, ValueError)):
            ops.q4_prefill_paged(lay, *args)
    free, cnt, qsl, st = z(9, dt=i32), z(1, dt=i32), z(4, dt=i32), z(5, dt=i64)
    for args in ((bt.long(), sq, qsl, free, cnt, 16, st), (bt, sq[:2], qsl, free, cnt, 16, st), (bt, sq, qsl[:3], free, cnt, 16, st),
                 (bt, sq, qsl, free[::2], cnt, 16, st), (bt, sq, qsl, free, z(2, dt=i32), 16, st), (bt, sq, qsl, free, cnt, 16, st.int()),
                 (bt, sq, qsl.cpu(), free, cnt, 16, st), (bt[:1].expand(3, 4), sq, qsl, free, cnt, 16, st)):
        with pytest.raises((TypeError, ValueError)):
            ops.plan_step(*args)
    with pytest.raises(ValueError):
        ops.plan_step(bt, sq, qsl, free, cnt, 16, st, positions=st[:2])
    with pytest.raises((TypeError, ValueError)):
        ops.release_blocks(bt, sq.cpu(), free, cnt, 16)
    from vllm_ttkv import _lib
    with pytest.raises(_lib.TTKVError):
        ops.release_blocks(bt, sq, free, cnt, 0)
