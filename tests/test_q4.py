"""The 4-bit cache's layout, the C entries' refusals (all before any launch: no GPU is needed) and the
oracle's own consistency."""
import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import q4 as O
from vllm_ttkv import _lib, ops
from vllm_ttkv.q4 import Q4Layout


def test_layout():
    lay = Q4Layout(H=8)
    assert (lay.panel_bytes, lay.bytes_per_token()) == (2176, 1088)
    assert abs(lay.ratio() - 4096 / 1088) < 1e-12
    assert lay.cache_shape(5, 64) == (5, 8, 4, 2176)
    cache = lay.new_cache(3, 32, device="cpu")
    assert lay.block_size(cache) == 32
    for d, g in ((64, 32), (64, 64), (128, 32), (128, 64), (128, 128)):
        assert Q4Layout(H=1, d=d, group=g).panel_bytes == O.panel_bytes(d, g) == _lib.lib().ttkv_q4_panel_bytes(d, g)
    for d, g in ((96, 32), (128, 16), (64, 128), (128, 48)):
        assert _lib.lib().ttkv_q4_panel_bytes(d, g) == 0
        with pytest.raises(ValueError):
            Q4Layout(H=1, d=d, group=g)
    with pytest.raises(ValueError):
        Q4Layout(H=0)
    for bs in (0, 8, 24):
        with pytest.raises(ValueError):
            lay.cache_shape(1, bs)
    for bad in (cache[0], cache.int(), cache[:, :4], cache[..., :16], cache.transpose(0, 1)):
        with pytest.raises(ValueError):
            lay.block_size(bad)


def test_ops_run_only_on_the_gpu():
    lay = Q4Layout(H=1, d=64, group=32)
    cache = lay.new_cache(2, 16, device="cpu")
    x = torch.zeros(1, 1, 64)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.q4_write_paged(lay, cache, torch.zeros(1, dtype=torch.int64), x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.q4_read_paged(lay, cache, torch.zeros(1, dtype=torch.int64), x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.q4_decode_paged(lay, cache, i32[None], i32, x.half(), 1.0, x.half())
    with pytest.raises(ValueError, match="CUDA"):
        ops.q4_prefill_paged(lay, cache, i32[None], i32, i32, i32, x.half(), 1.0, x.half(), 1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.plan_step(i32[None], i32, torch.zeros(2, dtype=torch.int32), i32, i32, 16, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.release_blocks(i32[None], i32, i32, i32, 16)


# stand-ins for device addresses: the calls below are refused before anything is launched
A = 1 << 20


CACHE = dict(base=A, n_blocks=4, H=2, d=128, group=64, block_size=16, flags=0)
STORE = CACHE | dict(slots=A, k=A, v=A, k_stride=256, v_stride=256, n=4, k_dtype=2, v_dtype=2, status=A, stream=0)
ATTN = CACHE | dict(block_table=A, seq_lens=A, q_start=A, q_len=A, q=A, out=A, bt_stride=4, q_stride=512, out_stride=512,
                    bt_cols=4, n_reqs=3, n_rows=9, HQ=4, dtype=2, max_q_len=3, max_seq_len=9, scale=1.0, workspace=A,
                    workspace_bytes=1 << 30, status=A, stream=0)
PLAN = dict(block_table=A, lens=A, query_start_loc=A, free_blocks=A, free_count=A, free_count_out=A, slots=A, positions=A,
            bt_stride=8, bt_cols=8, n_reqs=3, capacity=50, block_size=16, n_tokens=9, status=A, stream=0)


def _call(fn, cls, fields):
    """A C entry on a struct filled by name."""
    a = cls()
    for f, v in fields.items():
        setattr(a if hasattr(a, f) else a.cache, f, v)
    return fn(C.byref(a))


def _store(fn, **kw):
    return _call(fn, _lib.Q4StoreArgs, STORE | kw)


def _attn(fn, **kw):
    return _call(fn, _lib.Q4AttnArgs, ATTN | kw)


def _plan(fn, **kw):
    return _call(fn, _lib.PlanArgs, PLAN | kw)


BAD_CACHES = [(dict(d=96), _lib.ERR_UNSUPPORTED), (dict(group=16), _lib.ERR_UNSUPPORTED),
              (dict(d=64, group=128), _lib.ERR_UNSUPPORTED), (dict(block_size=8), _lib.ERR_UNSUPPORTED),
              (dict(block_size=40), _lib.ERR_UNSUPPORTED), (dict(H=0), _lib.ERR_ARG), (dict(base=0), _lib.ERR_ARG),
              (dict(n_blocks=-1), _lib.ERR_ARG), (dict(base=A + 8), _lib.ERR_ALIGN), (dict(H=70000), _lib.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches(kw, code):
    L = _lib.lib()
    assert _store(L.ttkv_q4_write, **kw) == code
    assert _store(L.ttkv_q4_read, **kw) == code
    assert _attn(L.ttkv_q4_decode, **kw) == code
    assert _attn(L.ttkv_q4_prefill, **kw) == code
    assert L.ttkv_last_error()


def test_store_refusals():
    L = _lib.lib()
    for kw, code in ((dict(slots=0), _lib.ERR_ARG), (dict(n=-1), _lib.ERR_ARG), (dict(k=0), _lib.ERR_ARG),
                     (dict(k_dtype=3), _lib.ERR_ARG), (dict(k_stride=255), _lib.ERR_ARG), (dict(v_dtype=-1), _lib.ERR_ARG),
                     (dict(v_stride=0), _lib.ERR_ARG), (dict(k=A + 1), _lib.ERR_ALIGN),
                     (dict(v=A + 2, v_dtype=0), _lib.ERR_ALIGN)):
        for fn in (L.ttkv_q4_write, L.ttkv_q4_read):
            assert _store(fn, **kw) == code, kw
            assert fn(None) == _lib.ERR_ARG
    assert _store(L.ttkv_q4_write, n=0, slots=0, k=0, v=0) == _lib.OK          # nothing to do


def test_attention_refusals():
    L = _lib.lib()
    ws = L.ttkv_q4_decode_workspace_bytes(128, 3, 2)
    wp = [L.ttkv_q4_prefill_workspace_bytes(128, 3, 2, n) for n in (3, 64)]
    assert ws > 0 and min(wp) > 0
    both = ((dict(q=0), _lib.ERR_ARG), (dict(out=0), _lib.ERR_ARG), (dict(dtype=0), _lib.ERR_UNSUPPORTED),
            (dict(q_stride=-1), _lib.ERR_ARG), (dict(out_stride=-8), _lib.ERR_ARG), (dict(HQ=3), _lib.ERR_ARG),
            (dict(HQ=1), _lib.ERR_ARG), (dict(workspace=0), _lib.ERR_WORKSPACE), (dict(workspace=A + 4), _lib.ERR_ALIGN),
            (dict(q=A + 1), _lib.ERR_ALIGN), (dict(block_table=0), _lib.ERR_ARG), (dict(seq_lens=0), _lib.ERR_ARG),
            (dict(n_reqs=-1), _lib.ERR_ARG), (dict(bt_cols=-1), _lib.ERR_ARG), (dict(n_reqs=70000), _lib.ERR_UNSUPPORTED),
            (dict(scale=float("nan")), _lib.ERR_ARG), (dict(scale=-float("inf")), _lib.ERR_ARG))
    for fn, extra in ((L.ttkv_q4_decode, {}), (L.ttkv_q4_prefill, {}), (L.ttkv_q4_prefill, dict(max_q_len=64))):
        for kw, code in both:
            assert _attn(fn, **(extra | kw)) == code, kw
        assert _attn(fn, n_reqs=0, **extra) == _lib.OK
        assert fn(None) == _lib.ERR_ARG
    assert _attn(L.ttkv_q4_decode, workspace_bytes=ws - 1) == _lib.ERR_WORKSPACE
    for n, need in zip((3, 64), wp):
        assert _attn(L.ttkv_q4_prefill, max_q_len=n, workspace_bytes=need - 1) == _lib.ERR_WORKSPACE
    for kw in (dict(q_start=0), dict(q_len=0), dict(max_q_len=-1), dict(max_seq_len=-1), dict(n_rows=-1)):
        assert _attn(L.ttkv_q4_prefill, **kw) == _lib.ERR_ARG, kw
    assert _attn(L.ttkv_q4_prefill, max_q_len=2 ** 30) == _lib.ERR_UNSUPPORTED
    assert _attn(L.ttkv_q4_prefill, n_rows=0) == _lib.OK


def test_plan_refusals():
    L = _lib.lib()
    both = ((dict(block_table=0), _lib.ERR_ARG), (dict(bt_stride=7), _lib.ERR_ARG), (dict(bt_cols=-1), _lib.ERR_ARG),
            (dict(lens=0), _lib.ERR_ARG), (dict(n_reqs=-1), _lib.ERR_ARG), (dict(free_blocks=0), _lib.ERR_ARG),
            (dict(capacity=-1), _lib.ERR_ARG), (dict(free_count=0), _lib.ERR_ARG), (dict(free_count_out=0), _lib.ERR_ARG),
            (dict(block_size=0), _lib.ERR_ARG), (dict(block_size=-16), _lib.ERR_ARG),
            (dict(n_reqs=_lib.PLAN_MAX_REQS + 1), _lib.ERR_UNSUPPORTED))
    for fn in (L.ttkv_plan_step, L.ttkv_release_blocks):
        for kw, code in both:
            assert _plan(fn, **kw) == code, kw
        assert fn(None) == _lib.ERR_ARG
    for kw in (dict(query_start_loc=0), dict(slots=0), dict(n_tokens=-1)):
        assert _plan(L.ttkv_plan_step, **kw) == _lib.ERR_ARG, kw


def test_structs_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ttkv_b200.h"', "int main(void) {"]
    structs = {"ttkv_q4_cache_t": _lib.Q4Cache, "ttkv_q4_store_args_t": _lib.Q4StoreArgs,
               "ttkv_q4_attn_args_t": _lib.Q4AttnArgs, "ttkv_plan_args_t": _lib.PlanArgs}
    for name, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    lines += ['printf("%d\\n", TTKV_PLAN_MAX_REQS);', "return 0;", "}"]
    src = tmp_path / "q4.c"
    src.write_text("\n".join(lines))
    subprocess.run([cc, "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "q4")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "q4")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in structs.values():
        want += [C.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want + [_lib.PLAN_MAX_REQS]


def test_oracle_quantises_within_half_a_scale():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)) * 10.0 ** rng.uniform(-2, 4, (50, 1))
    for g in (32, 64, 128):
        c, s, m = O.quantise(x, g)
        step = s.astype(np.float64).repeat(g, -1)
        # half a step, and what rounding the scale and the minimum to fp16 moves
        slack = 0.5 * step + 15 * step * 2.0 ** -11 + np.abs(m.astype(np.float64)).repeat(g, -1) * 2.0 ** -11
        assert np.all(np.abs(O.values(c, s, m) - x) <= slack)
