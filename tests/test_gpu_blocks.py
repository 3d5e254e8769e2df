"""Block tables and slot maps built on the GPU, against the oracle's plan request by request. Integers:
everything is equal."""
import numpy as np
import pytest
import torch

from oracle import q4 as O

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _run(table, seq, qsl, free, count, bs, T, positions=True, in_place=False):
    from vllm_ttkv import ops
    t, f, c = _i32(table), _i32(free), _i32([count])
    slots = torch.full((T,), 77, dtype=torch.int64, device="cuda")
    pos = torch.full((T,), 77, dtype=torch.int64, device="cuda") if positions else None
    co = None if in_place else _i32([-5])
    ops.plan_step(t, _i32(seq), _i32(qsl), f, c, bs, slots, positions=pos, free_count_out=co)
    got = c if in_place else co
    assert np.array_equal(f.cpu().numpy(), free)
    return t.cpu().numpy(), slots.cpu().numpy(), pos.cpu().numpy() if positions else None, int(got)


def _batch(rng, n, q_hi, hi, bs, cols, spare):
    seq = rng.integers(0, hi + 1, n)
    ql = np.minimum(rng.integers(0, q_hi + 1, n), seq)
    held = -(-(seq - ql) // bs)
    need = -(-seq // bs) - held
    total = int(held.sum() + need.sum()) + 40
    perm = rng.permutation(total)
    table = np.full((n, cols), -7, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = perm[at:at + h]
        at += h
    k = max(0, int(need.sum()) + spare)
    free = np.concatenate([perm[at:at + k], np.full(9, -3)])
    return table, seq, np.concatenate([[0], np.cumsum(ql)]), free, k


@pytest.mark.parametrize("n,q_hi,hi,bs", [(1, 1, 1, 16), (1, 500, 900, 16), (7, 1, 200, 1), (64, 1, 3000, 16), (513, 40, 300, 32),
                                          (1500, 3, 50, 17), (2048, 2, 40, 16), (2049, 2, 40, 16), (16384, 1, 20, 16)])
@pytest.mark.parametrize("pad", [0, 13])
def test_plan(n, q_hi, hi, bs, pad):
    rng = np.random.default_rng(n + bs)
    table, seq, qsl, free, count = _batch(rng, n, q_hi, hi, bs, -(-hi // bs) + 1, 5)
    T = int(qsl[-1]) + pad
    want = O.plan(table, seq, qsl, free, count, bs, T)
    assert not want[4]
    from vllm_ttkv import ops
    ops.reset_status()
    for in_place in (False, True):
        got = _run(table, seq, qsl, free, count, bs, T, positions=not in_place, in_place=in_place)
        ops.check_status()
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and got[3] == want[3]
        if not in_place:
            assert np.array_equal(got[2], want[2])


@pytest.mark.parametrize("spare", [-1, -20, -10 ** 6])
def test_plan_runs_out_of_blocks(spare):
    from vllm_ttkv import ops
    rng = np.random.default_rng(3)
    table, seq, qsl, free, count = _batch(rng, 200, 30, 300, 16, 20, spare)
    T = int(qsl[-1])
    want = O.plan(table, seq, qsl, free, count, 16, T)
    assert want[4]
    ops.reset_status()
    got = _run(table, seq, qsl, free, count, 16, T)
    with pytest.raises(RuntimeError, match="free list"):
        ops.check_status()
    assert all(np.array_equal(a, b) for a, b in zip(got[:3], want[:3])) and got[3] == want[3]


@pytest.mark.parametrize("what", ["more new tokens than tokens", "row too short", "tokens outside", "falling starts"])
def test_plan_refuses_a_request(what):
    from vllm_ttkv import ops
    table = np.full((4, 4), -7, np.int64)
    seq, ql = np.array([20, 30, 16, 5]), [20, 30, 16, 5]
    qsl = np.concatenate([[0], np.cumsum(ql)])
    T, free = 80, np.arange(100, 130)
    if what == "more new tokens than tokens":
        seq[1] = 29
    elif what == "row too short":
        seq[1], table = 65, np.where(np.arange(4) < 3, 50 + np.arange(4), table)
    elif what == "tokens outside":
        T = 70
    else:
        qsl = np.array([0, 20, 20, 19, 30])
        seq = np.array([20, 0, 5, 16])
    want = O.plan(table, seq, qsl, free, 20, 16, T)
    assert len(want[4]) == 1
    ops.reset_status()
    got = _run(table, seq, qsl, free, 20, 16, T)
    with pytest.raises(RuntimeError):
        ops.check_status()
    assert np.array_equal(got[0], want[0]) and got[3] == want[3]
    if what != "falling starts":                         # (there two requests share token 19)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])


def test_plan_without_requests_or_tokens():
    from vllm_ttkv import ops
    got = _run(np.zeros((0, 3)), np.zeros(0), [0], np.arange(5), 5, 16, 4)
    assert got[1].tolist() == [-1] * 4 and got[2].tolist() == [0] * 4 and got[3] == 5
    got = _run(np.full((2, 3), 9), [5, 0], [0, 0, 0], np.arange(5), 5, 16, 0)
    assert got[0].tolist() == [[9] * 3] * 2 and got[3] == 5
    ops.check_status()


@pytest.mark.parametrize("n,hi,bs", [(1, 1, 16), (5, 400, 16), (700, 90, 32)])
def test_release(n, hi, bs):
    from vllm_ttkv import ops
    rng = np.random.default_rng(n)
    lens = rng.integers(-1, hi + 1, n)
    nb = [max(0, -(-int(x) // bs)) for x in lens]
    cols = max(nb) + 1
    ids = rng.permutation(n * cols).reshape(n, cols)
    free = np.concatenate([np.arange(9) + 10 ** 6, np.full(sum(nb) + 3, -1)])
    want = free.copy()
    want[9:9 + sum(nb)] = np.concatenate([ids[r, :k] for r, k in enumerate(nb)])
    f, c = _i32(free), _i32([9])
    ops.reset_status()
    ops.release_blocks(_i32(ids), _i32(lens), f, c, bs)
    ops.check_status()
    assert int(c) == 9 + sum(nb) and np.array_equal(f.cpu().numpy(), want)


def test_release_refuses_what_does_not_fit():
    from vllm_ttkv import ops
    ids = np.arange(12).reshape(3, 4)
    free = np.full(8, -1)
    f, c = _i32(free), _i32([3])
    ops.reset_status()
    ops.release_blocks(_i32(ids), _i32([40, 48, 3]), f, c, 16)          # 3 + 3 + 1 blocks into 5 places
    with pytest.raises(RuntimeError, match="released"):
        ops.check_status()
    assert int(c) == 6 and f.cpu().tolist() == [-1] * 3 + [0, 1, 2] + [-1] * 2
    ops.release_blocks(_i32(ids), _i32([0, 65, 0]), f, c, 16)            # longer than its row
    with pytest.raises(RuntimeError):
        ops.check_status()
    assert int(c) == 6


def test_plan_captured():
    """A captured plan takes the lengths of each replay and moves the list on."""
    from vllm_ttkv import ops
    table = _i32(np.full((3, 8), -1))
    seq, qsl = _i32([1, 1, 0]), _i32([0, 1, 2, 2])
    free, count = _i32(np.arange(30)), _i32([30])
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int64, device="cuda")
    ops.status_word()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.plan_step(table, seq, qsl, free, count, 16, slots, positions=pos)
    ref, c = table.cpu().numpy().astype(np.int64), 30
    for i in range(40):
        seq.copy_(_i32([1 + i, 1 + i, 0]))
        g.replay()
        ref, s, p, c, bad = O.plan(ref, [1 + i, 1 + i, 0], [0, 1, 2, 2], np.arange(30), c, 16, 4)
        assert not bad
        assert np.array_equal(table.cpu().numpy(), ref) and slots.tolist() == s.tolist()
        assert pos.tolist() == p.tolist() and int(count) == c
    ops.check_status()


# ------------------------------------------------------------------ ids that are none
def _release(table, lens, free, count, bs):
    from vllm_ttkv import ops
    f, c = _i32(free), _i32([count])
    ops.release_blocks(_i32(table), _i32(lens), f, c, bs)
    return f.cpu().tolist()[:int(c)]


@pytest.mark.parametrize("n,hi", [(1, 40), (5, 400), (40, 5000), (700, 90), (5000, 40)])
def test_release_refuses_a_row_that_holds_no_id(n, hi):
    """A request with a negative id among its blocks returns none of them, the others all of theirs; one
    behind its blocks does not matter."""
    from vllm_ttkv import ops
    rng = np.random.default_rng(n)
    lens = rng.integers(1, hi + 1, n)
    nb = -(-lens // 16)
    cols = int(nb.max()) + 1
    table = rng.permutation(n * cols).reshape(n, cols)
    table[np.arange(n), nb] = -1
    for r in rng.permutation(n)[:max(1, n // 9)]:
        table[r, rng.integers(0, nb[r])] = -1 - int(rng.integers(0, 3))
    free = np.concatenate([np.arange(9) + 10 ** 6, np.full(int(nb.sum()), -1)])
    want, refused = O.release(table, lens, free, 9, 16)
    assert refused
    ops.reset_status()
    got = _release(table, lens, free, 9, 16)
    with pytest.raises(IndexError):
        ops.check_status()
    assert got == want and min(got) >= 0


def test_release_of_bad_rows_and_little_room():
    """The room of a refused request goes to those behind it; what does not fit even so is refused."""
    from vllm_ttkv import ops
    table = np.array([[1, -1, 3], [4, 5, 6], [7, 8, 9], [10, 11, 12], [-1, -1, -1]])
    for room, want in ((6, [4, 5, 6, 7, 8, 9]), (5, [4, 5, 6]), (8, [4, 5, 6, 7, 8, 9]), (9, [4, 5, 6, 7, 8, 9, 10, 11, 12])):
        free = np.full(room, -1)
        assert O.release(table, [48, 48, 48, 48, 0], free, 0, 16)[0] == want
        ops.reset_status()
        assert _release(table, [48, 48, 48, 48, 0], free, 0, 16) == want
        with pytest.raises((IndexError, RuntimeError)):
            ops.check_status()
    # one that would not fit and holds none: those behind it do
    free = np.full(5, -1)
    want = O.release(table[:3], [48, 32, 48], free, 3, 16)[0]
    assert want == [-1, -1, -1, 4, 5]
    ops.reset_status()
    assert _release(table[:3], [48, 32, 48], free, 3, 16) == want
    with pytest.raises((IndexError, RuntimeError)):
        ops.check_status()
    ops.reset_status()
    assert _release(table[1:], [33, 0, 48, 0], np.full(6, -1), 0, 16) == [4, 5, 6, 10, 11, 12]
    ops.check_status()


def test_a_refused_request_is_released():
    """A request that a step refused: released with the length it was planned with it is refused again, and
    nothing of its row reaches the list; released with the length it had, it returns what it held."""
    from vllm_ttkv import ops
    table = _i32([[3, 4, -7, -7], [5, 0, 1, 2], [-7, -7, -7, -7]])
    free, count = _i32([9, 8, -1, -1, -1, -1, -1]), _i32([2])
    slots = torch.zeros(60, dtype=torch.int64, device="cuda")
    ops.reset_status()
    ops.plan_step(table, _i32([33, 47, 0]), _i32([0, 1, 41, 41]), free, count, 16, slots)     # 1 block, then 2 of 1
    with pytest.raises(RuntimeError):
        ops.check_status()
    assert table.cpu().tolist()[:2] == [[3, 4, 8, -7], [5, -1, -1, 2]] and int(count) == 1
    ops.release_blocks(table, _i32([0, 47, 0]), free, count, 16)
    with pytest.raises(IndexError):
        ops.check_status()
    assert int(count) == 1 and int(free[0]) == 9
    ops.release_blocks(table, _i32([33, 7, 0]), free, count, 16)
    ops.check_status()
    assert free.cpu().tolist()[:int(count)] == [9, 3, 4, 8, 5]
    ops.plan_step(table, _i32([0, 0, 80]), _i32([0, 0, 0, 80]), free, count, 16, torch.zeros(80, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError):                    # (four columns)
        ops.check_status()
    ops.plan_step(table, _i32([0, 0, 60]), _i32([0, 0, 0, 60]), free, count, 16, slots)
    ops.check_status()
    assert table[2].tolist() == [5, 8, 4, 3] and int(count) == 1 and int(slots.min()) >= 0


def test_plan_reports_an_id_that_is_none():
    from vllm_ttkv import ops
    table, slots = _i32([[-7, -7], [-7, -7]]), torch.zeros(40, dtype=torch.int64, device="cuda")
    ops.reset_status()
    ops.plan_step(table, _i32([20, 20]), _i32([0, 20, 40]), _i32([4, 3, -1, 2]), _i32([4]), 16, slots)
    with pytest.raises(IndexError):
        ops.check_status()
    assert table.tolist() == [[2, -1], [3, 4]]
    assert slots.tolist() == [32 + i for i in range(16)] + [-1] * 4 + [48 + i for i in range(16)] + [64 + i for i in range(4)]


def test_release_captured():
    """A captured release, replayed with a row that holds no id and without."""
    from vllm_ttkv import ops
    table, lens = _i32([[1, 2], [3, 4], [5, 6]]), _i32([0, 0, 0])
    free, count, left = _i32(np.full(8, -1)), _i32([0]), _i32([-5])
    ops.status_word()
    ops.reset_status()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.release_blocks(table, lens, free, count, 16, free_count_out=left)
    for ns, row, want in (([20, 1, 0], [3, 4], [1, 2, 3]), ([20, 1, 32], [-1, 4], [1, 2, 5, 6]), ([0, 32, 1], [3, 4], [3, 4, 5]),
                          ([0, 32, 1], [3, -1], [5])):
        lens.copy_(_i32(ns))
        table[1].copy_(_i32(row))
        g.replay()
        assert free.tolist()[:int(left)] == want and int(count) == 0
        if min(row) < 0:
            with pytest.raises(IndexError):
                ops.check_status()
        else:
            ops.check_status()


def test_a_step_after_a_refusal_meets_no_other_blocks():
    """A request that was refused and whose next steps count its tokens as stored: its row holds ids that another
    request left there, and no token of it gets a slot in them."""
    from vllm_ttkv import ops
    bs, left = 16, [7, 6, 5, 4, 3, 2]                    # another request's blocks by now
    for first, new in ((20, 60), (1, 90), (16, 17)):
        table = _i32([[9] + left[1:]])
        if first > bs:
            table[0, 1] = 8
        free, count, slots = _i32([1, 0]), _i32([1]), torch.zeros(96, dtype=torch.int64, device="cuda")
        ops.reset_status()
        ops.plan_step(table, _i32([first + new]), _i32([0, new]), free, count, bs, slots)
        with pytest.raises(RuntimeError):
            ops.check_status()
        assert bool((slots == -1).all()) and int(count) == 1
        n = first + new
        while n < 96:
            n += 1
            ops.plan_step(table, _i32([n]), _i32([0, 1]), free, count, bs, slots[:1])
            if int(slots[0]) >= 0:                       # a block of its own, taken for this token or one before
                assert int(slots[0]) // bs == 1
        ops.reset_status()


def test_refused_rows_against_the_oracle():
    from vllm_ttkv import ops
    rng = np.random.default_rng(5)
    for _ in range(20):
        table, seq, qsl, free, count = _batch(rng, 60, 40, 300, 16, 20, -int(rng.integers(1, 60)))
        table = table[:, :int(rng.integers(15, 21))]
        T = int(qsl[-1]) - int(rng.integers(0, 3)) * 7
        want = O.plan(table, seq, qsl, free, count, 16, T)
        ops.reset_status()
        got = _run(table, seq, qsl, free, count, 16, T)
        with pytest.raises(RuntimeError):
            ops.check_status()
        assert all(np.array_equal(a, b) for a, b in zip(got[:3], want[:3])) and got[3] == want[3]
