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


def _cache(**kw):
    f = dict(base=A, n_blocks=4, H=2, d=128, group=64, block_size=16, flags=0) | kw
    return _lib.Q4Cache(*(f[n] for n, _ in _lib.Q4Cache._fields_))


def _batch(**kw):
    f = dict(block_table=A, bt_stride=4, bt_cols=4, seq_lens=A, n_reqs=3) | kw
    return _lib.Q4Batch(*(f[n] for n, _ in _lib.Q4Batch._fields_))


BAD_CACHES = [(dict(d=96), _lib.ERR_UNSUPPORTED), (dict(group=16), _lib.ERR_UNSUPPORTED),
              (dict(d=64, group=128), _lib.ERR_UNSUPPORTED), (dict(block_size=8), _lib.ERR_UNSUPPORTED),
              (dict(block_size=40), _lib.ERR_UNSUPPORTED), (dict(H=0), _lib.ERR_ARG), (dict(base=None), _lib.ERR_ARG),
              (dict(n_blocks=-1), _lib.ERR_ARG), (dict(base=A + 8), _lib.ERR_ALIGN), (dict(H=70000), _lib.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches(kw, code):
    L, c, b = _lib.lib(), C.byref(_cache(**kw)), C.byref(_batch())
    assert L.ttkv_q4_write(c, A, 1, A, 2, 256, A, 2, 256, A, None) == code
    assert L.ttkv_q4_read(c, A, 1, A, 2, 256, A, 2, 256, A, None) == code
    assert L.ttkv_q4_decode(c, b, A, 2, 512, 4, 1.0, A, 512, A, 1 << 30, A, None) == code
    assert L.ttkv_q4_prefill(c, b, A, A, A, 2, 512, 9, 4, 1.0, A, 512, 3, 9, A, 1 << 30, A, None) == code
    assert L.ttkv_last_error()


def test_store_refusals():
    L, c = _lib.lib(), C.byref(_cache())
    ok = [A, 4, A, 2, 256, A, 2, 256]
    for i, v, code in ((0, None, _lib.ERR_ARG), (1, -1, _lib.ERR_ARG), (2, None, _lib.ERR_ARG), (3, 3, _lib.ERR_ARG),
                       (4, 255, _lib.ERR_ARG), (6, -1, _lib.ERR_ARG), (7, 0, _lib.ERR_ARG), (2, A + 1, _lib.ERR_ALIGN)):
        args = list(ok)
        args[i] = v
        for fn in (L.ttkv_q4_write, L.ttkv_q4_read):
            assert fn(c, *args, A, None) == code, (i, v)
    assert L.ttkv_q4_write(None, *ok, A, None) == _lib.ERR_ARG
    assert L.ttkv_q4_write(c, A, 4, A + 2, 0, 256, A, 2, 256, A, None) == _lib.ERR_ALIGN
    assert L.ttkv_q4_write(c, None, 0, None, 2, 256, None, 2, 256, A, None) == _lib.OK       # nothing to do


def test_attention_refusals():
    L, c = _lib.lib(), C.byref(_cache())
    ws = L.ttkv_q4_decode_workspace_bytes(c, 3, 4)
    assert ws > 0
    ok = [A, 2, 512, 4, 1.0, A, 512, A, ws]
    for i, v, code in ((0, None, _lib.ERR_ARG), (1, 0, _lib.ERR_UNSUPPORTED), (2, -1, _lib.ERR_ARG), (3, 3, _lib.ERR_ARG),
                       (3, 1, _lib.ERR_ARG), (5, None, _lib.ERR_ARG), (6, -8, _lib.ERR_ARG), (7, None, _lib.ERR_WORKSPACE),
                       (8, ws - 1, _lib.ERR_WORKSPACE), (7, A + 4, _lib.ERR_ALIGN), (0, A + 1, _lib.ERR_ALIGN)):
        args = list(ok)
        args[i] = v
        assert L.ttkv_q4_decode(c, C.byref(_batch()), *args, A, None) == code, (i, v)
    for kw, code in ((dict(block_table=None), _lib.ERR_ARG), (dict(seq_lens=None), _lib.ERR_ARG), (dict(n_reqs=-1), _lib.ERR_ARG),
                     (dict(bt_cols=-1), _lib.ERR_ARG), (dict(n_reqs=70000), _lib.ERR_UNSUPPORTED)):
        assert L.ttkv_q4_decode(c, C.byref(_batch(**kw)), *ok, A, None) == code, kw
    assert L.ttkv_q4_decode(c, None, *ok, A, None) == _lib.ERR_ARG
    assert L.ttkv_q4_decode(c, C.byref(_batch(n_reqs=0)), *ok, A, None) == _lib.OK
    b = C.byref(_batch())
    ws = L.ttkv_q4_prefill_workspace_bytes(c, 3, 4, 64, 100)
    for args in ((None, A, 64, 100), (A, None, 64, 100), (A, A, -1, 100), (A, A, 64, -1)):
        assert L.ttkv_q4_prefill(c, b, args[0], args[1], A, 2, 512, 99, 4, 1.0, A, 512, args[2], args[3], A, ws, A, None) == _lib.ERR_ARG
    assert L.ttkv_q4_prefill(c, b, A, A, A, 2, 512, 0, 4, 1.0, A, 512, 64, 100, A, ws, A, None) == _lib.OK


def test_plan_refusals():
    L = _lib.lib()
    ok = [A, 8, 8, A, A, 3, A, 50, A, A, 16, A, A, 9]
    for i, v, code in ((0, None, _lib.ERR_ARG), (1, 7, _lib.ERR_ARG), (2, -1, _lib.ERR_ARG), (3, None, _lib.ERR_ARG),
                       (4, None, _lib.ERR_ARG), (5, -1, _lib.ERR_ARG), (6, None, _lib.ERR_ARG), (7, -1, _lib.ERR_ARG),
                       (8, None, _lib.ERR_ARG), (9, None, _lib.ERR_ARG), (10, 0, _lib.ERR_ARG), (11, None, _lib.ERR_ARG),
                       (13, -1, _lib.ERR_ARG), (5, _lib.PLAN_MAX_REQS + 1, _lib.ERR_UNSUPPORTED)):
        args = list(ok)
        args[i] = v
        assert L.ttkv_plan_step(*args, A, None) == code, (i, v)
    ok = [A, 8, 8, A, 3, A, 50, A, A, 16]
    for i, v, code in ((0, None, _lib.ERR_ARG), (3, None, _lib.ERR_ARG), (5, None, _lib.ERR_ARG), (7, None, _lib.ERR_ARG),
                       (8, None, _lib.ERR_ARG), (9, -16, _lib.ERR_ARG), (4, _lib.PLAN_MAX_REQS + 1, _lib.ERR_UNSUPPORTED)):
        args = list(ok)
        args[i] = v
        assert L.ttkv_release_blocks(*args, A, None) == code, (i, v)


def test_structs_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "ttkv_b200.h"', "int main(void) {"]
    structs = {"ttkv_q4_cache_t": _lib.Q4Cache, "ttkv_q4_batch_t": _lib.Q4Batch}
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
