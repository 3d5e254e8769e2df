"""What the attention over the 4-bit cache keeps of its precision where values are hard: tokens that some
rows of a block do not see, NaN beside numbers. The helpers, and the tolerances' terms, are those of
`test_gpu_q4.py`."""
import numpy as np
import pytest
import torch

from oracle import q4 as O
from q4_bounds import bound, worst
from test_gpu_q4 import DT, GEOMETRIES, _check_rows, _filled, _lay, _np, _prefill

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ drafted tokens that earlier rows do not see
def _small_values(lay, n, last, bs=16):
    """One request of n tokens, V of about 1e-3 but for `last` [k, H, d], the V of the last k tokens:
    (cache, table, K, V stored)."""
    from vllm_ttkv import ops
    rng = np.random.default_rng(n)
    nb = -(-n // bs)
    cache = lay.new_cache(nb, bs)
    table = torch.from_numpy(rng.permutation(nb)).int()[None].cuda()
    t = torch.arange(n, device="cuda")
    k = torch.from_numpy(rng.standard_normal((n, lay.H, lay.d))).float().cuda()
    v = torch.from_numpy(rng.standard_normal((n, lay.H, lay.d)) * 1e-3).float().cuda()
    v[n - len(last):] = last
    ops.q4_write_paged(lay, cache, table[0].long()[t // bs] * bs + t % bs, k, v)
    return cache, table, *(O.values(*O.quantise(_np(x), lay.group)) for x in (k, v))


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("G,ql,n", [(1, 5, 70), (2, 4, 64), (4, 6, 203), (3, 8, 1000)])
@pytest.mark.parametrize("what", ["nan", "large", "infinite lane"])
def test_a_later_token_costs_earlier_rows_nothing(d, g, G, ql, n, what):
    """The last two tokens' V are NaN or 10^7 times the others': the rows before them, of the same block and the
    same unit of tokens, are as exact as without them."""
    lay = _lay(1, d, g)
    last = torch.full((2, 1, d), float("nan") if what == "nan" else 3e4, device="cuda")
    if what == "large":
        last *= torch.linspace(0.5, 1, d, device="cuda")
    if what == "infinite lane":
        last = torch.full((2, 1, d), 1e-3, device="cuda")
        last[..., 5] = float("inf")
    cache, table, K, V = _small_values(lay, n, last)
    q = torch.randn(ql, G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, d ** -0.5, out)
    _check_rows(_np(out[:-2]), _np(q[:-2]), K[:n - 2], V[:n - 2], d ** -0.5, G, torch.float16, False)
    if what == "large":
        _check_rows(_np(out[-2:]), _np(q[-2:]), K, V, d ** -0.5, G, torch.float16, False)
    else:                                                # the lanes of the groups that hold one, and no other
        spoilt = torch.zeros(d, dtype=torch.bool)
        spoilt[:d if what == "nan" else g] = True
        assert bool(out[-2:, :, spoilt.cuda()].isnan().all())
        if g < d and what != "nan":
            rest = ~spoilt.numpy()
            got, want = _np(out[-2:])[..., rest], O.attend(_np(q[-2:]), K, np.where(np.isnan(V), 0, V), d ** -0.5, G)[..., rest]
            R = np.nanmax(np.abs(V))
            assert np.all(np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2 * 2.0 ** -12 * R)


@pytest.mark.parametrize("d,g", [(64, 32), (128, 128)])
def test_a_bad_block_of_the_last_rows_costs_the_others_nothing(d, g):
    from vllm_ttkv import ops
    lay, n, ql, G = _lay(1, d, g), 66, 6, 2
    cache, table, K, V = _small_values(lay, n, torch.full((2, 1, d), 1e-3, device="cuda"))
    table[0, -1] = cache.shape[0] + 3                    # tokens 64 and 65: the last two queries
    q = torch.randn(ql, G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    ops.reset_status()
    _prefill(lay, cache, table, [n], [ql], q, d ** -0.5, out)
    with pytest.raises(IndexError):
        ops.check_status()
    assert bool(out[-2:].isnan().all())
    _check_rows(_np(out[:-2]), _np(q[:-2]), K[:n - 2], V[:n - 2], d ** -0.5, G, torch.float16, False)


@pytest.mark.parametrize("d,g", GEOMETRIES)
def test_scales_that_rise_and_parts_that_meet(d, g):
    """V scales that grow along the tokens, over parts of several CTAs, with rows that end in different units."""
    lay, n, ql, G = _lay(2, d, g), 5003, 9, 2
    from vllm_ttkv import ops
    rng = np.random.default_rng(7)
    nb = -(-n // 16)
    cache = lay.new_cache(nb, 16)
    table = torch.from_numpy(rng.permutation(nb)).int()[None].cuda()
    t = torch.arange(n, device="cuda")
    k = torch.from_numpy(rng.standard_normal((n, 2, d))).float().cuda()
    v = torch.from_numpy(rng.standard_normal((n, 2, d)) * np.exp2(np.linspace(-14, 6, n))[:, None, None]).float().cuda()
    v[n - 7::2] *= 500
    ops.q4_write_paged(lay, cache, table[0].long()[t // 16] * 16 + t % 16, k, v)
    K, V = (O.values(*O.quantise(_np(x), g)) for x in (k, v))
    q = torch.randn(ql, 2 * G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, d ** -0.5, out)
    for j in range(ql):                                  # row by row: R is what the row itself sees
        m = n - ql + j + 1
        _check_rows(_np(out[j:j + 1]), _np(q[j:j + 1]), K[:m], V[:m], d ** -0.5, G, torch.float16, False)


# ------------------------------------------------------------------ NaN in chunks
@pytest.mark.parametrize("d,g", [(64, 32), (128, 128)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_nan_by_row_tiles_in_turn(d, g, dtype):
    """Row blocks of two row tiles and of one in turn, many in a CTA: a NaN of V in a block's last tokens reaches
    the rows that see it, and the rows of no other block."""
    from vllm_ttkv import ops
    lay, R, G, n0 = _lay(1, d, g), 700, 4, 300
    qls = [60 if r % 2 else 20 for r in range(R)]        # 240 and 80 rows
    seqs = [n0 - 10 + r % 40 for r in range(R)]
    # every request reads one of eight stored sequences; in the odd ones a token near the end is NaN
    cache, table, K, V = _filled(lay, [n0 + 40] * 8, 16, seed=d)
    at = [seqs[-1] - 12 - 3 * i for i in range(8)]
    for i in range(1, 8, 2):
        one = torch.zeros(1, 1, d, device="cuda")
        bad = one.clone()
        bad[..., 1] = float("nan")
        ops.q4_write_paged(lay, cache, table[i, at[i] // 16].long()[None] * 16 + at[i] % 16, one, bad)
        K[i][at[i]] = 0.0
    own = [(r * 3) % 8 for r in range(R)]
    q = torch.randn(sum(qls), G, d, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.empty_like(q)
    ops.reset_status()
    starts = _prefill(lay, cache, table[torch.tensor(own, device="cuda")].contiguous(), seqs, qls, q, d ** -0.5, out, max_q=100)
    ops.check_status()
    nan = out.isnan().cpu().numpy()
    for r in range(R):
        i, a, ql, n = own[r], starts[r], qls[r], seqs[r]
        sees = (n - ql + np.arange(ql)) >= at[i] if i % 2 else np.zeros(ql, bool)
        assert np.array_equal(nan[a:a + ql, :, :g].all((1, 2)), sees) and np.array_equal(nan[a:a + ql, :, :g].any((1, 2)), sees), r
        assert not nan[a:a + ql, :, g:].any(), r
        if r % 50 < 3:
            clean = V[i].copy()
            clean[at[i]] = 0.0 if i % 2 else clean[at[i]]
            got, ref = _np(out[a:a + ql]), _np(q[a:a + ql])
            if sees.any():
                got[sees, :, :g] = O.attend(ref, K[i][:n], clean[:n], d ** -0.5, G)[sees, :, :g]
            _check_rows(got, ref, K[i][:n], clean[:n], d ** -0.5, G, DT[dtype], True)


# ------------------------------------------------------------------ small weights beside a large one
@pytest.mark.parametrize("d,g", [(64, 64), (128, 128)])
@pytest.mark.parametrize("R,ql,n", [(1, 1, 16384), (160, 1, 4000), (1, 66, 50000), (160, 33, 16384)])
@pytest.mark.parametrize("nats", [8, 13, 17, 18, 20])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_token_that_takes_most(d, g, R, ql, n, nats, dtype):
    """The first token's weight is e^nats times each other's, and its value is 0: the output is what the many small
    weights carry. Keys, values and queries lie on grids that fp16 holds, so that nothing is rounded but
    weights, sums and the output, in chunks as well. Tolerance: half a step of the output; 2^-11 of each
    weight, which acts on the value or on half its group's range, and 2^-12 of the same for what is in fp32;
    and 2^-30 of the largest weight in each, where fp16 has no bits left. Few requests (a row in parts, of
    which one holds the first token) and many (rows whole)."""
    from vllm_ttkv import ops
    lay, G = _lay(1, d, g), 2
    rng = np.random.default_rng(ql)
    nb = -(-n // 16)
    cache, table = lay.new_cache(nb, 16), torch.from_numpy(rng.permutation(nb)).int()[None].cuda()
    k, v = (rng.integers(-7, 9, (n, 1, d)) / 8.0 for _ in range(2))
    for x in (k, v):                                     # every group's codes go from 0 to 15
        x[:, :, ::g], x[:, :, 1::g] = -7 / 8, 1.0
    v[1:, :, 2:] = np.abs(v[1:, :, 2:])
    v[0] = 0.0
    k[0] = np.where(np.arange(d) % 2, 1.0, -7 / 8)
    t = torch.arange(n, device="cuda")
    kt, vt = (torch.from_numpy(x).float().cuda() for x in (k, v))
    ops.q4_write_paged(lay, cache, table[0].long()[t // 16] * 16 + t % 16, kt, vt)
    K, V = (O.values(*O.quantise(x, g)) for x in (k, v))
    assert np.array_equal(K, k) and np.array_equal(V, v)
    q = torch.from_numpy(np.where(np.arange(d) % 2, 1.0, -1.0) * np.ones((ql, G, 1))).to(DT[dtype]).cuda()
    s = (K[:, 0] @ q[0, 0].double().cpu().numpy())       # the first is the largest of all
    scale = nats / (s[0] - np.median(s[1:]))
    out = torch.empty(R * ql, G, d, device="cuda", dtype=DT[dtype])
    _prefill(lay, cache, table.expand(R, -1), [n] * R, [ql] * R, q.repeat(R, 1, 1), scale, out)
    want = O.attend(_np(q), K, V, scale, G)
    W = np.maximum(np.abs(V), np.where(np.arange(n) > 0, 7.5 / 8, 0.0)[:, None, None])
    tol = torch.finfo(DT[dtype]).eps / 2 * np.abs(want) + (2.0 ** -11 + 2.0 ** -12) * O.attend(_np(q), K, W, scale, G) + n * 2.0 ** -30
    err = np.abs(_np(out).reshape(R, ql, G, d) - want)
    assert np.all(err <= tol), (float((err / tol).max()), float((err / np.abs(want).max()).max()))


# ------------------------------------------------------------------ queries of no number
@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("ql,G", [(1, 2), (5, 3), (140, 2)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_an_infinite_query_is_nan(d, g, ql, G, sign, scale):
    """Keys of one sign in the lane that the query is infinite in, and groups whose least value has that sign or
    not: all the scores are then +inf or all -inf, and the formula's answer is NaN."""
    from vllm_ttkv import ops
    lay, n = _lay(1, d, g), ql + 70
    rng = np.random.default_rng(ql)
    cache, table = lay.new_cache(-(-n // 16), 16), torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
    k, v = (torch.from_numpy(rng.uniform(0.5, 2, (n, 1, d))).float().cuda() for _ in range(2))
    ops.q4_write_paged(lay, cache, torch.arange(n, device="cuda"), k, v)
    K, V = (O.values(*O.quantise(_np(x), g)) for x in (k, v))
    q = torch.randn(ql, G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    q[ql // 2, 1, 7] = sign * float("inf")
    out = torch.empty_like(q)
    if ql == 1:
        ops.q4_decode_paged(lay, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), q, scale, out)
    else:
        _prefill(lay, cache, table, [n], [ql], q, scale, out)
    assert bool(out[ql // 2, 1].isnan().all())
    got, ref = _np(out), _np(q)
    ref[ql // 2, 1] = 0.0
    got[ql // 2, 1] = O.attend(ref, K, V, scale, G)[ql // 2, 1]
    _check_rows(got, ref, K, V, scale, G, torch.float16, True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_an_infinite_query_of_a_long_row_is_nan(dtype):
    """As above, the row in parts of many CTAs, some of them behind what the row sees."""
    lay, n, ql = _lay(1, 64, 64), 3000, 200
    from vllm_ttkv import ops
    rng = np.random.default_rng(1)
    cache, table = lay.new_cache(-(-n // 16), 16), torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
    k, v = (torch.from_numpy(rng.uniform(0.5, 2, (n, 1, 64))).float().cuda() for _ in range(2))
    ops.q4_write_paged(lay, cache, torch.arange(n, device="cuda"), k, v)
    q = torch.randn(ql, 2, 64, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    q[11, 0, 7] = q[150, 1, 40] = -float("inf")
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, 0.1, out)
    want = torch.zeros(ql, 2, dtype=torch.bool)
    want[11, 0] = want[150, 1] = True
    nan = out.isnan().cpu()
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)


def test_lengths_next_to_32_bits_are_refused():
    """A row of 2048 blocks of 2^20 tokens: longer requests than a 32-bit position behind their last tile allows are
    refused on the device, the others served."""
    from vllm_ttkv import ops
    lay, bs = _lay(1, 64, 64), 2 ** 20
    cache = lay.new_cache(1, bs)
    table = torch.zeros(3, 2048, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2))
    ops.q4_write_paged(lay, cache, torch.arange(40, device="cuda"), k, v)
    K, V = (O.values(*O.quantise(_np(x), 64)) for x in (k, v))
    for n in (2 ** 31 - 255, 2 ** 31 - 60, 2 ** 31 - 1):
        for ql, G in ((1, 2), (2, 4), (100, 4)):
            q = torch.randn(3 * ql, G, 64, generator=torch.Generator().manual_seed(3)).half().cuda()
            out = torch.full_like(q, 5.0)
            seqs = [40, n, 40]
            ops.reset_status()
            if ql == 1:
                ops.q4_decode_paged(lay, cache, table, torch.tensor(seqs, dtype=torch.int32, device="cuda"), q, 0.1, out)
            else:
                _prefill(lay, cache, table, seqs, [min(ql, 40), ql, min(ql, 40)], q, 0.1, out, max_q=ql)
            with pytest.raises(RuntimeError, match="seq_len"):
                ops.check_status()
            m = min(ql, 40)
            assert bool((out[m:m + ql] == 5).all())
            for a in (0, m + ql):
                _check_rows(_np(out[a:a + m]), _np(q[a:a + m]), K, V, 0.1, G, torch.float16, True)


# ------------------------------------------------------------------ chunks, tile by tile
def _check_tight(out, q, K, V, scale, G, lay, chunk):
    w = worst(_np(out), *bound(_np(q), K, V, scale, G, torch.finfo(out.dtype).eps / 2, lay.group, chunk))
    assert w <= 1, w


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("H,HQ,dtype,bs", [(1, 1, "fp16", 16), (2, 6, "bf16", 16), (1, 13, "fp16", 64), (2, 16, "fp16", 32)])
@pytest.mark.parametrize("qls", [(100, 127, 128, 129), (300, 0, 33, 65), (1, 257, 2, 90)])
def test_chunks(d, g, H, HQ, dtype, bs, qls):
    """Every query is as exact as its operands allow: a stored tile that is lost or stale, or a limit that is off
    by a token, would show (`test_q4_bounds.py`)."""
    lay = _lay(H, d, g)
    seqs = [n + extra if n else 0 for n, extra in zip(qls, (0, 130, 5, 333))]
    cache, table, K, V = _filled(lay, seqs, bs, seed=HQ + d)
    q = torch.randn(sum(qls), HQ, d, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.full_like(q, 5.0)
    starts = _prefill(lay, cache, table, seqs, qls, q, d ** -0.5, out)
    for r, (a, n) in enumerate(zip(starts, qls)):
        if n:
            _check_tight(out[a:a + n], q[a:a + n], K[r], V[r], d ** -0.5, HQ // H, lay, True)


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("scale,dtype", [(0.05, "fp16"), (0.2, "fp16"), (0.05, "bf16")])
def test_chunks_of_many_tiles(d, g, scale, dtype):
    """Some 40 stored tiles a CTA, many times round the ring of panels and the operands' stages."""
    lay, R, ql, n, G = _lay(1, d, g), 64, 64, 6000, 8
    cache, table, K, V = _filled(lay, [n], 16, seed=d + g)
    q = torch.randn(R * ql, G, d, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table.expand(R, -1), [n - 3 * r for r in range(R)], [ql] * R, q, scale, out)
    for r in (0, 11, 23, 38, 47, 63):
        a, m = starts[r], n - 3 * r
        _check_tight(out[a:a + ql], q[a:a + ql], K[0][:m], V[0][:m], scale, G, lay, True)


@pytest.mark.parametrize("H,HQ,ql,n", [(1, 2, 200, 5000), (2, 8, 40, 3001), (1, 16, 9, 9000), (1, 5, 700, 2100)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_chunks_in_parts(H, HQ, ql, n, dtype):
    lay = _lay(H, 128, 128)
    cache, table, K, V = _filled(lay, [n], 16, seed=ql)
    q = torch.randn(ql, HQ, 128, generator=torch.Generator().manual_seed(3)).to(DT[dtype]).cuda()
    out = torch.empty_like(q)
    _prefill(lay, cache, table, [n], [ql], q, 0.08, out)
    _check_tight(out, q, K[0], V[0], 0.08, HQ // H, lay, True)


@pytest.mark.parametrize("d,g", GEOMETRIES)
@pytest.mark.parametrize("R,H,G,ql,n", [(5, 2, 3, 1, 1031), (40, 1, 4, 4, 300), (7, 2, 4, 6, 2000), (3, 1, 8, 3, 700), (1, 1, 5, 4, 9000)])
def test_few_rows(d, g, R, H, G, ql, n):
    """At most 24 rows of a KV head: streamed, with keys and values as they are stored."""
    lay = _lay(H, d, g)
    seqs = [ql + int(x) for x in np.random.default_rng(R).integers(0, n, R)]
    seqs[0] = n
    cache, table, K, V = _filled(lay, seqs, 16, seed=R)
    q = torch.randn(R * ql, G * H, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table, seqs, [ql] * R, q, d ** -0.5, out)
    for r, a in enumerate(starts):
        _check_tight(out[a:a + ql], q[a:a + ql], K[r], V[r], d ** -0.5, G, lay, False)


@pytest.mark.parametrize("d,g", [(128, 32), (128, 128)])
@pytest.mark.parametrize("ql,G", [(7, 4), (8, 4), (3, 11)])
def test_rows_next_to_the_choice_of_kernel(d, g, ql, G):
    """25 to 33 rows of a KV head over long rows, which go to one kernel or the other by the groups."""
    lay, R = _lay(1, d, g), 40
    seqs = [1400 + 7 * r for r in range(R)]
    cache, table, K, V = _filled(lay, [max(seqs)], 16, seed=R)
    q = torch.randn(R * ql, G, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    out = torch.empty_like(q)
    starts = _prefill(lay, cache, table.expand(R, -1), seqs, [ql] * R, q, d ** -0.5, out)
    for r in range(0, R, 9):
        a, m = starts[r], seqs[r]
        streamed = g > 32 and ql * G <= 32
        _check_tight(out[a:a + ql], q[a:a + ql], K[0][:m], V[0][:m], d ** -0.5, G, lay, not streamed)


# ------------------------------------------------------------------ calls one behind the other
def test_a_chain_of_calls_without_a_pause():
    """Plan, write, read back, attend and release, each of which may start while the one before it runs: the same
    bits as with the device waited for after every call."""
    from vllm_ttkv import ops
    lay, bs, R, HQ, T = _lay(2, 64, 32), 16, 24, 8, 24 * 40
    rng = np.random.default_rng(3)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    steps, lens = [], np.zeros(R, np.int64)
    for step in range(30):
        done = (rng.uniform(size=R) < 0.15) & (lens > 0)
        gone = np.where(done, lens, 0)
        lens = np.where(done, 0, lens)
        new = np.where(lens == 0, rng.integers(1, 41, R), 1 if step % 3 else rng.integers(1, 9, R))
        lens = lens + new
        kv = [torch.from_numpy(rng.standard_normal((T, 2, 64))).half().cuda() for _ in range(2)]
        steps.append((i32(gone), i32(lens), i32(np.concatenate([[0], np.cumsum(new)])), i32(np.cumsum(new) - new), i32(new),
                      *kv, torch.from_numpy(rng.standard_normal((T, HQ, 64))).half().cuda(), int(new.max()), int(lens.max())))

    def run(pause):
        cache = lay.new_cache(400, bs)
        table = torch.full((R, 30), -1, dtype=torch.int32, device="cuda")
        free, count = torch.arange(400, dtype=torch.int32, device="cuda"), i32([400])
        slots, pos = (torch.zeros(T, dtype=torch.int64, device="cuda") for _ in range(2))
        outs = []
        torch.cuda.synchronize()
        for gone, ln, qsl, qs, ql, k, v, q, max_q, max_n in steps:
            out, dec, ko, vo = (torch.zeros_like(x) for x in (q, q[:R], k, v))
            for call in (lambda: ops.release_blocks(table, gone, free, count, bs),
                         lambda: ops.plan_step(table, ln, qsl, free, count, bs, slots, positions=pos),
                         lambda: ops.q4_write_paged(lay, cache, slots, k, v, skip_pad=True),
                         lambda: ops.q4_read_paged(lay, cache, slots, ko, vo, skip_pad=True),
                         lambda: ops.q4_write_paged(lay, cache, slots, ko, vo, skip_pad=True),
                         lambda: ops.q4_prefill_paged(lay, cache, table, ln, qs, ql, q, 0.125, out, max_q, max_n),
                         lambda: ops.q4_decode_paged(lay, cache, table, ln, out[:R], 0.125, dec)):
                call()
                if pause:
                    torch.cuda.synchronize()
            outs += [out, dec, ko, vo, slots.clone(), table.clone(), free[:10].clone()]
        ops.check_status()
        return outs

    ops.reset_status()
    want = run(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
