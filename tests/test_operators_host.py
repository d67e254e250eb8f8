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


def test_extents_meet_where_their_bytes_do(tmp_path):
    """The host's rule for what two tensors of a call share, against sets of bytes."""
    (tmp_path / "x.cpp").write_text("""
        #include "extent.h"
        #include <set>
        #include <random>
        #include <cstdio>
        using namespace ts;
        static std::set<uintptr_t> bytes(uintptr_t p, uint64_t b, uint64_t s, uint64_t n) {
            std::set<uintptr_t> r;
            for (uint64_t i = 0; i < n; ++i) for (uint64_t j = 0; j < b; ++j) r.insert(p + i * s + j);
            return r;
        }
        int main() {
            std::mt19937 g(1);
            auto in = [&](int lo, int hi) { return lo + (int)(g() % (hi - lo + 1)); };
            int met = 0;
            for (int k = 0; k < 200000; ++k) {
                uint64_t b[2], s[2], n[2]; uintptr_t p[2];
                for (int i = 0; i < 2; ++i) { b[i] = in(0, 6); n[i] = in(0, 5); s[i] = b[i] + (in(0, 2) ? in(0, 12) : 0); p[i] = in(1, 60); }
                if (in(0, 1)) s[1] = s[0] < b[1] ? b[1] : s[0];
                auto x = bytes(p[0], b[0], s[0], n[0]), y = bytes(p[1], b[1], s[1], n[1]);
                bool want = false;
                for (auto v : x) want = want || y.count(v);
                met += want;
                if (overlap(Extent((void*)p[0], b[0], s[0], n[0]), Extent((void*)p[1], b[1], s[1], n[1])) != want) {
                    printf("%d: %d %d %d %d, %d %d %d %d\\n", k, (int)p[0], (int)b[0], (int)s[0], (int)n[0], (int)p[1], (int)b[1], (int)s[1], (int)n[1]);
                    return 1;
                }
            }
            return met > 20000 && met < 180000 ? 0 : 2;
        }""")
    subprocess.check_call(["g++", "-std=c++17", "-I", build.CSRC, str(tmp_path / "x.cpp"), "-o", str(tmp_path / "x")])
    subprocess.check_call([str(tmp_path / "x")])


NOWHERE = 1 << 20                # no such device: what is not refused before ends there (3), and nothing is launched


def _far(**kw):
    """Pointers far apart from each other."""
    return {name: (i + 1) << 32 for i, name in enumerate(kw.pop("names").split())} | kw


def test_calls_refuse_outputs_that_share_memory(lib):
    def norm(**kw):
        return lib.ts_norm_rotate(C.byref(_norm(device=NOWHERE, **(_far(names="q k positions q_weight k_weight q_out k_out k_plain") | kw))))
    p = _far(names="q k positions q_weight k_weight q_out k_out k_plain")
    row = 4 * 128 * 2                                                         # bytes of a token's queries; of its keys half
    assert norm() == 3
    assert norm(q_out=p["q"]) == norm(k_out=p["k"]) == norm(k_plain=p["k"]) == norm(q_out=p["q"], k_out=p["k"]) == 3          # in place
    for shift in (2, row, 2 * row, -2, -2 * row):
        assert norm(q_out=p["q"] + shift) == 1
    assert norm(q_out=p["q"] + 3 * row) == norm(q_out=p["q"] - 3 * row) == 3
    assert norm(q_out=p["q"], q_stride=1024) == norm(q_out=p["q"] + row, q_stride=1024) == 1 and norm(q_out=p["q"], q_stride=1024, tokens=1) == 3
    assert norm(q_out=p["q"] + row, q_stride=5 * 512) == 3 and norm(q_out=p["q"] + row, q_stride=4 * 512 - 8) == 1            # the gap behind a token
    for bad in (dict(q_out=p["k"]), dict(k_out=p["q"] + 8), dict(k_plain=p["q"] + row), dict(k_plain=p["k"] + 256), dict(k_out=p["k"] + 256),
                dict(q_out=p["k_out"] - row), dict(k_plain=p["k_out"]), dict(k_plain=p["q_out"] + 8), dict(k_out=p["positions"]), dict(q_out=p["k_weight"] - 8)):
        assert norm(**bad) == 1, bad

    names = "q k v cu_seqlens out"
    p = _far(names=names)

    def call(**kw):
        return lib.ts_prompt_attend(C.byref(_prompt(device=NOWHERE, **(p | kw))))
    assert call() == 3 and call(k=p["q"], v=p["q"]) == 3
    out = 10 * row
    for x, stride in (("q", 512), ("k", 256), ("v", 1024)):
        end = ((9 * stride) + (512 if x == "q" else 256)) * 2
        assert call(out=p[x]) == call(out=p[x] + 16) == call(out=p[x] + end - 16) == call(out=p[x] - out + 16) == 1
        assert call(out=p[x] + end) == call(out=p[x] - out) == 3
    assert call(out=p["cu_seqlens"] - 16) == 1 and call(out=p["cu_seqlens"] + 16) == 3

    p = _far(names="k v rows pool")

    def rows(call, **kw):
        return call(C.byref(_rows(device=NOWHERE, **(p | kw))))
    half, pool = 1024 * 2, 10 * 8 * 144
    for c in (lib.ts_quant_write, lib.ts_quant_read):
        assert rows(c) == 3
        assert rows(c, k=p["v"] + half, k_stride=2048, v_stride=2048) == 3                               # K behind V in one buffer
        assert rows(c, k=p["pool"] + pool - 16) == rows(c, v=p["pool"] - 16) == rows(c, rows=p["pool"] + 4) == 1
        assert rows(c, k=p["pool"] + pool) == rows(c, v=p["pool"] - 4 * half) == 3
    assert rows(lib.ts_quant_write, k=p["v"]) == 3                                                       # reading the same rows twice is no harm
    assert rows(lib.ts_quant_read, k=p["v"]) == rows(lib.ts_quant_read, k=p["v"] + 2 * half) == rows(lib.ts_quant_read, k=p["v"] + half, k_stride=2047, v_stride=2048) == 1
    assert rows(lib.ts_quant_read, v=p["rows"] - 8) == 1

    p = _far(names="q pool req_to_token req_pool_indices seq_lens out workspace")
    for bad in ("pool", "req_to_token", "req_pool_indices", "seq_lens"):
        assert lib.ts_quant_attend(C.byref(_attend(device=NOWHERE, **(p | {"out": p[bad] + 4})))) == 1, bad
    assert lib.ts_quant_attend(C.byref(_attend(device=NOWHERE, **p))) == 3 == lib.ts_quant_attend(C.byref(_attend(device=NOWHERE, **(p | {"out": p["q"]}))))


def test_numbers_that_are_not_finite_are_refused(lib):
    """An infinite soft cap would make every logit undefined, an infinite base of the angles leave a pair unturned."""
    for x in (float("inf"), float("nan")):
        for bad in (dict(logit_cap=x), dict(sm_scale=x), dict(rope_base=x), dict(rope_scale=x)):
            assert lib.ts_quant_attend(C.byref(_attend(device=NOWHERE, **(_far(names="q pool req_to_token req_pool_indices seq_lens out workspace") | bad)))) == 1, bad
        for bad in (dict(logit_cap=x), dict(sm_scale=x)):
            assert lib.ts_prompt_attend(C.byref(_prompt(device=NOWHERE, **(_far(names="q k v cu_seqlens out") | bad)))) == 1, bad
        for bad in (dict(rope_base=x), dict(rope_scale=x)):
            p = _far(names="q k positions q_out k_out")
            assert lib.ts_norm_rotate(C.byref(_norm(device=NOWHERE, **(p | bad)))) == 1, bad
            assert lib.ts_norm_rotate(C.byref(_norm(device=NOWHERE, **(p | bad | {"positions": None})))) == 3, bad
    assert lib.ts_prompt_attend(C.byref(_prompt(device=NOWHERE, logit_cap=-1.0, **_far(names="q k v cu_seqlens out")))) == 3
