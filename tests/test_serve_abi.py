"""Serving operators' C-ABI (include/mtc_serve.h) without a GPU: every declared function is exported, the ctypes structs
mirror the C ones, and host-side checks turn bad arguments into error codes before any GPU call."""

import ctypes
import os
import re
import subprocess

import pytest

from tensorpack_amd import _abi, _native

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")


@pytest.fixture(scope="module")
def lib():
    return _native.hip_lib()


def test_every_declared_symbol_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(INCLUDE, "mtc_serve.h")).read(), flags=re.S)
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(mtc_[a-z_0-9]+)\s*\(", text, flags=re.M))
    assert names == set(_abi.SERVE_EXPORTED)
    assert all(hasattr(lib, n) for n in names)


def test_constants_and_struct_layouts_match_c(tmp_path):
    structs = {"mtc_heads": _abi.MtcHeads, "mtc_prompt_args": _abi.MtcPromptArgs, "mtc_cache_desc": _abi.MtcCacheDesc,
               "mtc_cached_args": _abi.MtcCachedArgs, "mtc_verify_args": _abi.MtcVerifyArgs}
    consts = {"MTC_DTYPE_F16": _abi.MTC_DTYPE_F16, "MTC_ATTN_MAX_DIM": _abi.ATTN_MAX_DIM, "MTC_CACHED_MAX_TOKENS": _abi.CACHED_MAX_TOKENS,
              "MTC_CACHED_MAX_SEQS": _abi.CACHED_MAX_SEQS, "MTC_CACHE_MAX_SLOTS": _abi.CACHE_MAX_SLOTS}
    src = "#include <stddef.h>\n#include <stdio.h>\n#include \"mtc_serve.h\"\nint main(void){\n"
    want = []
    for c, py in structs.items():
        src += f'printf("%zu\\n", sizeof({c}));\n'
        want.append(ctypes.sizeof(py))
        for f, _ in py._fields_:
            src += f'printf("%zu\\n", offsetof({c}, {f}));\n'
            want.append(getattr(py, f).offset)
    for c, v in consts.items():
        src += f'printf("%zu\\n", (size_t){c});\n'
        want.append(v)
    (tmp_path / "t.c").write_text(src + "return 0;}\n")
    subprocess.run(["gcc", "-I", INCLUDE, str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == want
    assert set(_abi.CACHE_STATUS) == {1, 2, 4, 8, 16}


def _heads(data=0x1000, row=512, head=64):
    return _abi.MtcHeads(data, row, head)


def _prompt(**kw):
    a = _abi.MtcPromptArgs(_abi.ABI_VERSION, _abi.MTC_DTYPE_BF16, 1, 8, 2, 64, 10, 10, 1, 0.125, _heads(), _heads(), _heads(), _heads(),
                           0x2000, 0x2000)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_prompt_checks(lib):
    f = lambda a, stream: lib.mtc_prompt_attention(a, None, 0, stream)
    assert f(None, None) == -1
    for kw, code in (({"abi_version": 3}, -7), ({"dtype": 0}, -4), ({"dtype": 9}, -4), ({"heads": 7}, -3), ({"kv_heads": 0}, -3),
                     ({"dim": 60}, -3), ({"dim": 136}, -3), ({"dim": 0}, -3), ({"scale": 0.0}, -3), ({"scale": float("inf")}, -3),
                     ({"n_seqs": -1}, -3), ({"q_rows": -1}, -3), ({"cu_q": None}, -1), ({"cu_k": None}, -1),
                     ({"q": _heads(None)}, -1), ({"k": _heads(0x1008)}, -3), ({"v": _heads(row=516)}, -3), ({"o": _heads(head=-64)}, -3),
                     ({"k": _heads(row=32)}, -3), ({"q": _heads(row=1 << 24)}, -3), ({"heads": 1 << 30, "kv_heads": 1}, -3)):
        assert f(_prompt(**kw), None) == code, kw
        assert lib.mtc_last_error()
    assert f(_prompt(n_seqs=0), None) == 0 and f(_prompt(q_rows=0), None) == 0
    ws, few = lib.mtc_prompt_attention_workspace_bytes, dict(q_rows=100, k_rows=5000)
    assert ws(_prompt()) == 0 and ws(_prompt(q_rows=100000, k_rows=100000)) == 0 and ws(_prompt(heads=7)) == 0
    need = ws(_prompt(**few))                                    # few rows on many keys: partial results
    assert need >= 2 * 100 * 8 * 66 * 4
    full = lib.mtc_prompt_attention
    assert full(_prompt(**few), None, need, None) == -5 and full(_prompt(**few), 0x100, need - 1, None) == -5
    assert full(_prompt(**few), 0x180, need, None) == -5


def _cache(**kw):
    c = _abi.MtcCacheDesc(_abi.ABI_VERSION, _abi.MTC_DTYPE_BF16, 100, 2, 2, 64, 16, 8, 10, 0, 0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def test_cache_checks(lib):
    assert lib.mtc_check_cache_desc(_cache()) == 0 and lib.mtc_check_cache_desc(None) == -1
    for kw, code in (({"abi_version": 1}, -7), ({"dtype": 0}, -4), ({"n_pages": 0}, -2), ({"n_layers": 0}, -2), ({"dim": 12}, -2),
                     ({"dim": 256}, -2), ({"page_size": 8}, -2), ({"page_size": 24}, -2), ({"page_size": 512}, -2),
                     ({"max_seqs": 1 << 17}, -2), ({"max_pages": 1 << 27}, -2), ({"pool": None}, -1), ({"pool": 0x1008}, -2),
                     ({"table": None}, -1), ({"scratch": None}, -1), ({"reserved": 1}, -2)):
        assert lib.mtc_check_cache_desc(_cache(**kw)) == code, kw
    assert lib.mtc_cache_scratch_ints(100, 8) == 308 and lib.mtc_cache_scratch_ints(0, 8) == 0
    c, p = _cache(), 0x7000
    assert lib.mtc_cache_extend(c, None, p, 1, None) == -1 and lib.mtc_cache_extend(c, p, None, 1, None) == -1
    assert lib.mtc_cache_extend(c, p, p, 9, None) == -3 and lib.mtc_cache_extend(c, p, p, -1, None) == -3
    assert lib.mtc_cache_extend(_cache(dim=12), p, p, 1, None) == -2
    assert lib.mtc_cache_fork(c, p, None, 1, None) == -1 and lib.mtc_cache_fork(c, p, p, 8193, None) == -3
    assert lib.mtc_cache_truncate(c, None, p, 1, None) == -1
    assert lib.mtc_cache_compact(_cache(page_size=8), None) == -2
    assert lib.mtc_cache_copy_pages(c, None, 5, p, p, 1, None) == -1 and lib.mtc_cache_copy_pages(c, 0x1000, 0, p, p, 1, None) == -3
    h = ctypes.byref(_heads())
    assert lib.mtc_cache_append(c, 2, h, h, 1, 1, p, p, 1, None) == -3 and lib.mtc_cache_append(c, 0, h, h, 2, 1, p, p, 1, None) == -4
    assert lib.mtc_cache_append(c, 0, h, h, 1, -1, p, p, 1, None) == -3 and lib.mtc_cache_append(c, 0, h, h, 1, 1, p, None, 1, None) == -1
    assert lib.mtc_cache_append(c, 0, ctypes.byref(_heads(0x1004)), h, 1, 1, p, p, 1, None) == -3
    for call in (lambda: lib.mtc_cache_extend(c, None, None, 0, None), lambda: lib.mtc_cache_fork(c, None, None, 0, None),
                 lambda: lib.mtc_cache_truncate(c, None, None, 0, None), lambda: lib.mtc_cache_copy_pages(c, None, 0, None, None, 0, None),
                 lambda: lib.mtc_cache_append(c, 0, h, h, 0, 0, None, None, 0, None)):
        assert call() == 0                                       # nothing to do


def _cached(**kw):
    a = _abi.MtcCachedArgs(_abi.ABI_VERSION, 1, 4, 2, 8, 0, 0.125, 0, _heads(), _heads(), 0x7000, None, None, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_cached_checks(lib):
    f, ws, c = lib.mtc_cached_attention, lib.mtc_cached_attention_workspace_bytes, _cache()
    need = ws(c, _cached())
    assert need > 0 and ws(c, _cached(n_groups=2)) > need
    for kw, code in (({"abi_version": 1}, -7), ({"layer": 2}, -3), ({"layer": -1}, -3), ({"n_seqs": 8193}, -3), ({"n_seqs": 9, "seqs": None}, -3),
                     ({"tokens": 0}, -3), ({"tokens": 17}, -3), ({"heads": 3}, -3), ({"scale": -1.0}, -3), ({"n_groups": 5}, -3),
                     ({"reserved": 1}, -3)):
        assert f(c, _cached(**kw), 0x100, 1 << 40, None) == code, kw
        assert ws(c, _cached(**kw)) == 0
    assert f(c, None, 0x100, need, None) == -1 and f(_cache(page_size=8), _cached(), 0x100, need, None) == -2
    assert f(c, _cached(), None, need, None) == -5 and f(c, _cached(), 0x100, need - 1, None) == -5
    assert f(c, _cached(), 0x80, need, None) == -5
    assert f(c, _cached(n_groups=1), 0x100, 1 << 40, None) == -1
    assert f(c, _cached(q=_heads(None)), 0x100, need, None) == -1 and f(c, _cached(o=_heads(0x1004)), 0x100, need, None) == -3
    assert f(c, _cached(n_seqs=0), None, 0, None) == 0


def _verify(**kw):
    two = (ctypes.c_int64 * 2)(400, 100)
    a = _abi.MtcVerifyArgs(_abi.ABI_VERSION, 0, 4, 2, 3, 100, 0x1000, two, 0x2000, two, 0x3000, 3, 0x4000, 100, 0x5000, 3, None, 0x6000, 0x7000)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_verify_checks(lib):
    f, ws = lib.mtc_verify_drafts, lib.mtc_verify_workspace_bytes
    need = ws(_verify())
    assert need > 0
    for kw, code in (({"abi_version": 1}, -7), ({"dtype": 3}, -4), ({"index_bytes": 2}, -4), ({"n_seqs": 65536}, -3), ({"n_drafted": 65}, -3),
                     ({"vocab": 0}, -3), ({"p": None}, -1), ({"q": None}, -1), ({"u": None}, -1), ({"noise": None}, -1), ({"drafts": None}, -1),
                     ({"tokens": None}, -1), ({"accepted": None}, -1)):
        assert f(_verify(**kw), 0x100, need, None) == code, kw
    assert f(None, 0x100, need, None) == -1 and f(_verify(), None, need, None) == -5 and f(_verify(), 0x100, need - 1, None) == -5
    assert f(_verify(), 0x104, need, None) == -5
    assert f(_verify(n_seqs=0), None, 0, None) == 0


def test_without_a_gpu_the_calls_raise():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    from tensorpack_amd.attention import prompt_attention
    from tensorpack_amd.cache import PagedCache
    from tensorpack_amd.sampling import verify_drafts
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        prompt_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError):
        PagedCache(8, 1, 2, 64, max_seqs=2, max_pages=4)
    with pytest.raises(RuntimeError):
        verify_drafts(torch.zeros(1, 1, dtype=torch.int32), *[torch.zeros(1, n, 8) for n in (2, 1)], torch.zeros(1, 1), torch.zeros(1, 8))
