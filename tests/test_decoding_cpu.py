"""CPU checks of the decoding operators (faiss_amd/decoding.py): what is refused before anything is launched, and the kernels'
registers.  Sizes and types are checked before the handle, so a null handle is the error of a call whose sizes are right."""
import ctypes
import os
import re
import sys

import pytest
import torch

import faiss_amd
from faiss_amd import decoding

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CACHE = dict(code=1, numBlocks=10, blockSize=16, numHeads=2, headDim=64)


def _error(fn, *args):
    lib = faiss_amd.load_library()
    assert getattr(lib, fn)(*args) == -2
    return lib.faiss_amd_get_last_error().decode()


def _cache(**kw):
    return decoding._CacheStruct(**{**CACHE, **kw})


def _attend(cache=None, **kw):
    a = decoding._AttendStruct(**{**dict(tableStride=4, batch=2, tokens=2, heads=4, numColumns=4, maxQueries=1, type=3, causal=1, scale=0.125), **kw})
    return _error("faiss_amd_PagedCache_attend", None, ctypes.byref(cache or _cache()), ctypes.byref(a), None)


@pytest.mark.parametrize("kw, say", [
    (dict(code=2), "code"), (dict(blockSize=8), "block size"), (dict(blockSize=48), "block size"), (dict(blockSize=512), "block size"),
    (dict(headDim=80), "head dimension"), (dict(headDim=512), "head dimension"), (dict(numHeads=0), "heads"),
    (dict(numBlocks=0), "blocks"), (dict(numBlocks=1 << 27), "blocks")])
def test_a_cache_of_another_kind_is_refused(kw, say):
    assert say in _attend(_cache(**kw))
    add = decoding._AddStruct(type=3, tokens=1)
    assert say in _error("faiss_amd_PagedCache_add", None, ctypes.byref(_cache(**kw)), ctypes.byref(add), None)
    assert say in _error("faiss_amd_PagedCache_reconstruct", None, ctypes.byref(_cache(**kw)), 1, None, 1, None, None, 0, None)


@pytest.mark.parametrize("kw, say", [
    (dict(), "null resources"), (dict(type=1), "float16 or bfloat16"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"),
    (dict(batch=-1), "negative"), (dict(tokens=3), "one query per request"), (dict(tableStride=3), "overlap"),
    (dict(numColumns=1 << 27, tableStride=1 << 27), "too wide"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite")])
def test_attend_refuses(kw, say):
    assert say in _attend(**kw)


def test_null_structs_are_errors():
    c = ctypes.byref(_cache())
    assert "null cache" in _error("faiss_amd_PagedCache_attend", None, None, None, None)
    assert "null arguments" in _error("faiss_amd_PagedCache_attend", None, c, None, None)
    assert "null arguments" in _error("faiss_amd_PagedCache_add", None, c, None, None)
    assert "null arguments" in _error("faiss_amd_plan_blocks", None, None, None)
    assert "null arguments" in _error("faiss_amd_beam_select", None, None, None)
    assert "null arguments" in _error("faiss_amd_fork_blocks", None, 1, c, None, None)
    assert "null output" in _error("faiss_amd_PagedCache_attend_workspace", None, c, None, None)
    assert "null output" in _error("faiss_amd_beam_select_workspace", None, None, None)


@pytest.mark.parametrize("kw, say", [
    (dict(), "null resources"), (dict(beams=0), "64"), (dict(beams=65), "64"), (dict(keep=0), "64"), (dict(keep=65), "64"),
    (dict(vocab=0), "vocabulary"), (dict(vocab=1 << 31), "vocabulary"), (dict(padToken=-1), "padToken"), (dict(padToken=100), "padToken"),
    (dict(type=0), "float32"), (dict(batch=-1), "negative")])
def test_beam_select_refuses(kw, say):
    a = decoding._BeamStruct(**{**dict(vocab=100, batch=1, beams=2, keep=2, type=1), **kw})
    assert say in _error("faiss_amd_beam_select", None, ctypes.byref(a), None)


@pytest.mark.parametrize("kw, say", [
    (dict(), "null resources"), (dict(batch=-1), "negative"), (dict(maxTokens=-1), "negative"), (dict(numBlocks=0), "blocks"),
    (dict(blockSize=0), "blocks"), (dict(numBlocks=1 << 28), "blocks"), (dict(tableStride=3), "overlap"),
    (dict(numColumns=1 << 28, tableStride=1 << 28), "too wide")])
def test_plan_blocks_refuses(kw, say):
    a = decoding._PlanStruct(**{**dict(tableStride=4, batch=2, numColumns=4, numBlocks=8, blockSize=16, maxTokens=3), **kw})
    assert say in _error("faiss_amd_plan_blocks", None, ctypes.byref(a), None)


def test_reorder_and_fork_refuse():
    assert "null resources" in _error("faiss_amd_reorder_beams", None, 1, None, None, 1, 2, 2, 0, None)
    assert "negative" in _error("faiss_amd_reorder_beams", None, -1, None, None, 1, 2, 2, 0, None)
    assert "negative" in _error("faiss_amd_reorder_beams", None, 1, None, None, 1, 0, 2, 0, None)
    fork = dict(tableStride=4, batch=1, beams=2, numColumns=4)
    two = (decoding._CacheStruct * 2)(_cache(), _cache(blockSize=32))
    for kw, n, c, say in ((dict(), 1, two, "null resources"), (dict(), 2, two, "different blocks"), (dict(), 0, two, "at least one"),
                          (dict(beams=0), 1, two, "negative"), (dict(tableStride=2), 1, two, "overlap")):
        a = decoding._ForkStruct(**{**fork, **kw})
        assert say in _error("faiss_amd_fork_blocks", None, n, c, ctypes.byref(a), None)


class _Res:  # what the wrappers look at before the library sees the call
    device = 0
    _h = None
    _lib = None


def test_wrappers_refuse_wrong_types_and_devices():
    i32, f32 = torch.int32, torch.float32
    t, n = torch.zeros((2, 4), dtype=i32), torch.zeros(2, dtype=i32)
    with pytest.raises(TypeError):
        decoding.plan_blocks(_Res, t.long(), n, n, n, n, 16, 3)
    with pytest.raises(ValueError):
        decoding.plan_blocks(_Res, n, n, n, n, n, 16, 3)
    with pytest.raises(ValueError, match="device"):
        decoding.plan_blocks(_Res, t, n, n, n, n, 16, 3)
    with pytest.raises(TypeError):
        decoding.beam_select(_Res, [1.0], t, 2)
    with pytest.raises(ValueError, match="device"):
        decoding.beam_select(_Res, torch.zeros((1, 2, 3)), torch.zeros((1, 2)), 2)
    with pytest.raises(ValueError, match="device"):
        decoding.reorder_beams(_Res, [], t)
    with pytest.raises(ValueError):
        decoding.PagedCache(_Res, 4, 16, 2, 64, code="int4")
    with pytest.raises(TypeError):
        decoding.PagedCache.wrap(_Res, torch.zeros((1, 1, 16, 64)), torch.zeros((1, 1, 64, 16)), torch.zeros((1, 1)), torch.zeros((1, 1)))


def test_the_structs_match_the_header():
    """field names and order of the ctypes structs against include/faiss_amd_c.h"""
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "faiss_amd_c.h")).read(), flags=re.S)
    for name, st in (("PagedCache", decoding._CacheStruct), ("PlanBlocksParams", decoding._PlanStruct), ("CacheAddParams", decoding._AddStruct),
                     ("AttendParams", decoding._AttendStruct), ("BeamSelectParams", decoding._BeamStruct), ("BeamState", decoding._StateStruct),
                     ("ForkBlocksParams", decoding._ForkStruct)):
        body = re.search(r"typedef struct FaissAmd%s \{(.*?)\}" % name, hdr, re.S).group(1)
        want = []
        for decl in body.split(";"):
            words = re.sub(r"\b(const|unsigned)\b", "", decl).strip()
            if words:
                kind, names = re.match(r"(\w+)\s*(.*)", words, re.S).groups()
                for x in names.split(","):
                    x = x.strip()
                    want.append((x.strip("* "), ctypes.c_void_p if "*" in x else
                                 {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "size_t": ctypes.c_size_t}[kind]))
        got = [(f.rstrip("_"), t) for f, t in st._fields_]
        assert got == want, name


@pytest.fixture(scope="module")
def builds(tmp_path_factory):
    sys.path.insert(0, os.path.join(ROOT, "tools"))
    import isa_lint
    if not os.path.exists(isa_lint.HIPCC):
        pytest.skip("hipcc not available")
    out = {}
    d = tmp_path_factory.mktemp("isa")
    for name in ("cache_attention.hip", "decoding_kernels.hip"):
        asm = str(d / (name + ".s"))
        err = isa_lint.compile_asm(os.path.join(isa_lint.CSRC, name), asm, extra=["-Rpass-analysis=kernel-resource-usage"])
        out[name] = (open(asm).read(), err)
    return out


def test_kernels_stay_in_registers(builds):
    """no scratch, no out-of-line call, no packed fp32 instruction, no LDS through generic pointers"""
    for name, (asm, remarks) in builds.items():
        assert "s_swappc_b64" not in asm and "src_shared_base" not in asm, name
        assert not re.search(r"v_pk_(add|mul|fma)_f32", asm), name
        scratch = re.findall(r"Function Name: (\S+).*?ScratchSize \[bytes/lane\]: (\d+)", remarks, re.S)
        assert scratch and all(int(s) == 0 for _, s in scratch), [x for x in scratch if int(x[1])]
