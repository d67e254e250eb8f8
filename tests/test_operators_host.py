"""CPU-only checks of the 4-bit cache, head-norm and packed-prompt calls: struct layouts, refusals, and the plain forms that
the GPU tests compare with.  No kernel is launched here."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from tests import operators_ref as ref
from tokenselect_b200 import _lib, build, prompt, quant_cache as qc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def test_struct_layouts_match_the_header(tmp_path):
    pairs = [("ts_quant_rows_args", _lib.TsQuantRowsArgs), ("ts_quant_attend_args", _lib.TsQuantAttendArgs),
             ("ts_norm_rotate_args", _lib.TsNormRotateArgs), ("ts_prompt_args", _lib.TsPromptArgs)]
    lines = "".join(f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {n}));' for n, _ in t._fields_) for c, t in pairs)
    (tmp_path / "s.c").write_text('#include "tokenselect_b200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){' + lines + "return 0;}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = list(map(int, subprocess.check_output([str(tmp_path / "s")]).split()))
    want = [x for _, t in pairs for x in (C.sizeof(t), *(getattr(t, n).offset for n, _ in t._fields_))]
    assert got == want


PTR = 1 << 20                    # never dereferenced: every call here is refused, or has nothing to do, before a launch


def _rows(**kw):
    a = dict(struct_size=C.sizeof(_lib.TsQuantRowsArgs), dtype=0, hkv=8, head_dim=128, count=4, k=PTR, v=PTR, k_stride=1024, v_stride=1024,
             rows=PTR, pool=PTR, pool_rows=10, k_scale=1.0, v_scale=1.0)
    return _lib.TsQuantRowsArgs(**{**a, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(struct_size=4), 1), (dict(dtype=2), 2), (dict(head_dim=96), 2), (dict(hkv=0), 1), (dict(hkv=1025), 1), (dict(count=-1), 1),
    (dict(pool_rows=0), 1), (dict(k_stride=1023), 1), (dict(v_stride=0), 1), (dict(k_scale=3.0), 1), (dict(v_scale=0.0), 1),
    (dict(k_scale=-1.0), 1), (dict(v_scale=float("nan")), 1), (dict(k_scale=2.0 ** 33), 1), (dict(k=None), 1), (dict(v=None), 1),
    (dict(rows=None), 1), (dict(pool=None), 1), (dict(pool=PTR + 8), 1), (dict(count=0, k=None, v=None, rows=None, pool=None), 0),
], ids=str)
def test_row_calls_refuse(lib, bad, status):
    for call in (lib.ts_quant_write, lib.ts_quant_read):
        assert call(C.byref(_rows(**bad))) == status
        assert call(None) == 1


def _attend(**kw):
    a = dict(struct_size=C.sizeof(_lib.TsQuantAttendArgs), dtype=0, batch=2, hq=32, hkv=8, head_dim=128, max_reqs=4, q=PTR, pool=PTR, pool_rows=10,
             req_to_token=PTR, req_to_token_stride=100, max_ctx=100, req_pool_indices=PTR, seq_lens=PTR, out=PTR, sm_scale=0.1, rope_base=1e4,
             rope_scale=1.0, k_scale=1.0, v_scale=1.0, workspace=PTR, workspace_bytes=1 << 40)
    return _lib.TsQuantAttendArgs(**{**a, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(struct_size=4), 1), (dict(dtype=7), 2), (dict(head_dim=256), 2), (dict(batch=-1), 1), (dict(batch=1025), 1), (dict(hq=30), 1),
    (dict(hq=72), 2), (dict(hkv=0), 1), (dict(rope_base=0.0), 1), (dict(rope_scale=-1.0), 1), (dict(k_scale=0.3), 1), (dict(sm_scale=0.0), 1),
    (dict(sm_scale=float("inf")), 1), (dict(sm_scale=float("nan")), 1), (dict(max_reqs=0), 1), (dict(max_ctx=-1), 1), (dict(max_ctx=1 << 40), 1),
    (dict(batch=1024, max_ctx=(1 << 31) - 100), 1), (dict(pool_rows=0), 1), (dict(pool=PTR + 4), 1), (dict(workspace=PTR + 4), 1),
    (dict(workspace=None), 1), (dict(q=None), 1), (dict(out=None), 1), (dict(seq_lens=None), 1), (dict(batch=0, q=None, out=None, workspace=None), 0),
], ids=str)
def test_attention_refuses(lib, bad, status):
    assert lib.ts_quant_attend(C.byref(_attend(**bad))) == status
    assert lib.ts_quant_attend(None) == 1
    n = C.c_size_t()
    assert lib.ts_quant_attend_workspace(0, 2000, 32, 128, C.byref(n)) == 1 and lib.ts_quant_attend_workspace(0, 1, 32, 96, C.byref(n)) == 2


def _norm(**kw):
    a = dict(struct_size=C.sizeof(_lib.TsNormRotateArgs), dtype=0, tokens=3, hq=4, hkv=2, head_dim=128, eps=1e-6, q=PTR, k=PTR, q_stride=512,
             k_stride=256, positions=PTR, rope_base=1e4, rope_scale=1.0, q_out=PTR, k_out=PTR)
    return _lib.TsNormRotateArgs(**{**a, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(struct_size=0), 1), (dict(dtype=9), 2), (dict(head_dim=80), 2), (dict(tokens=-1), 1), (dict(hq=0), 1), (dict(hkv=1025), 1),
    (dict(q_stride=511), 1), (dict(k_stride=100), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(rope_base=0.0), 1), (dict(q=None), 1),
    (dict(k_out=None), 1), (dict(tokens=0, q=None, k=None, q_out=None, k_out=None), 0),
], ids=str)
def test_norm_refuses(lib, bad, status):
    assert lib.ts_norm_rotate(C.byref(_norm(**bad))) == status
    assert lib.ts_norm_rotate(None) == 1


def _prompt(**kw):
    a = dict(struct_size=C.sizeof(_lib.TsPromptArgs), dtype=0, tokens=10, batch=2, hq=4, hkv=2, head_dim=128, sm_scale=0.1, q=PTR, k=PTR, v=PTR,
             q_stride=512, k_stride=256, v_stride=1024, cu_seqlens=PTR, out=PTR)
    return _lib.TsPromptArgs(**{**a, **kw})


@pytest.mark.parametrize("bad,status", [
    (dict(struct_size=0), 1), (dict(dtype=9), 2), (dict(head_dim=80), 2), (dict(tokens=-1), 1), (dict(batch=4097), 1), (dict(hq=5), 1),
    (dict(q_stride=500), 1), (dict(v_stride=8), 1), (dict(sm_scale=0.0), 1), (dict(sm_scale=-0.1), 1), (dict(k=None), 1), (dict(cu_seqlens=None), 1),
    (dict(q=PTR + 8), 1), (dict(k_stride=260), 1), (dict(dtype=1, k_stride=258), 1), (dict(out=PTR + 2), 1), (dict(tokens=0, q=None), 0),
    (dict(batch=0, cu_seqlens=None), 0),
], ids=str)
def test_prompt_attention_refuses(lib, bad, status):
    assert lib.ts_prompt_attend(C.byref(_prompt(**bad))) == status
    assert lib.ts_prompt_attend(None) == 1


def test_python_entry_points_refuse_what_the_kernels_would_misread():
    """There is no CPU path, and tensors of the wrong type, shape or layout do not reach the library."""
    i32 = torch.int32
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    pool, rows = qc.kv4_pool(10, 2, 128, device="cpu"), torch.zeros(4, dtype=i32)
    assert pool.shape == (10, 2, 144) and qc.kv4_row_bytes(64) == 72
    for p in (pool, pool.float(), pool[:, :, :100]):
        with pytest.raises(ValueError, match="pool"):
            qc.kv4_write(p, k, k, rows)
        with pytest.raises(ValueError, match="pool"):
            qc.kv4_read(p, rows)
        with pytest.raises(ValueError, match="pool"):
            qc.kv4_attend(k.view(4, 256), p, rows[None], rows, rows, 0.1, 1e4)
    with pytest.raises(ValueError, match="q must be"):
        prompt.norm_rotate(k, k, None)
    with pytest.raises(ValueError, match="q must be"):
        prompt.prompt_attend(k, k, k, rows, 0.1)


def test_plain_quantiser_is_the_nearest_level():
    """The reference form the GPU results are held to: no level is nearer, and a block's largest element keeps 6/7 of itself
    or more."""
    x = torch.randn(50, 2, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-2, 2, 50)[:, None, None]
    codes, scales = ref.quantise(x)
    got = ref.values(codes, scales)
    s = torch.tensor(ref.SCALES, dtype=torch.float64)[scales].repeat_interleave(16, -1)
    every = torch.tensor(ref.LEVELS, dtype=torch.float64)
    best = (x.double().abs()[..., None] - every * s[..., None]).abs().amin(-1)
    assert torch.equal((x.double() - got).abs(), best)
    pool = ref.pack(x, x.flip(0))
    a, b = ref.unpack(pool)
    assert torch.equal(a, got) and torch.equal(b, got.flip(0)) and pool.shape == (50, 2, 144)
    rel = ((x.double() - got).norm() / x.double().norm()).item()
    assert rel < 0.12


def test_plain_attention_skips_what_is_not_seen():
    q, k = torch.randn(3, 2, 64), torch.randn(3, 1, 64)
    v = torch.randn(3, 1, 64)
    v[2] = float("nan")
    seen = torch.tensor([[1, 0, 0], [1, 1, 0], [0, 0, 0]], dtype=torch.bool)
    o, mag = ref.attend(q, k, v, seen, 0.1)
    assert torch.allclose(o[0, 0], v[0, 0].double()) and torch.isfinite(o).all() and not o[2].any() and (mag >= o.abs() - 1e-12).all()
    assert torch.equal(ref.causal([1, 0, 2], 3), torch.tensor([[1, 0, 0], [0, 1, 0], [0, 1, 1]], dtype=torch.bool))
