"""CPU checks of what the decoding operators refuse before anything is launched: sizes past a launch, gradients, layouts that a
kernel cannot read.  Sizes and types are checked before the handle, so a null handle is the error of a call whose sizes are right."""
import ctypes

import pytest
import torch

import faiss_amd
from faiss_amd import decoding


def _error(fn, *args):
    lib = faiss_amd.load_library()
    assert getattr(lib, fn)(*args) == -2
    return lib.faiss_amd_get_last_error().decode()


def _cache(**kw):
    return decoding._CacheStruct(**{**dict(code=1, numBlocks=10, blockSize=16, numHeads=2, headDim=64), **kw})


# the largest sizes that launch, and the next: a launch holds less than 2^32 threads, and all of a call's are checked before the first
@pytest.mark.parametrize("batch, tokens, fits", [(2 ** 24 - 1, 0, True), (2 ** 24, 0, False), (2 ** 24 - 2, 1024, True), (2 ** 24 - 2, 1025, False),
                                                 (2 ** 24 - 2 ** 21 - 1, 2 ** 31 - 1, True), (2 ** 24 - 2 ** 21, 2 ** 31 - 1, False)])
def test_plan_blocks_past_a_launch(batch, tokens, fits):
    a = decoding._PlanStruct(tableStride=4, batch=batch, numColumns=4, numBlocks=8, blockSize=16, maxTokens=tokens)
    assert ("null resources" if fits else "too many rows") in _error("faiss_amd_plan_blocks", None, ctypes.byref(a), None)


@pytest.mark.parametrize("n, heads, fits", [(2 ** 24 - 1, 1, True), (2 ** 24, 1, False), (2 ** 23 - 1, 2, True), (2 ** 23, 2, False), (2 ** 31 - 1, 32767, False)])
def test_reconstruct_past_a_launch(n, heads, fits):
    say = _error("faiss_amd_PagedCache_reconstruct", None, ctypes.byref(_cache(numHeads=heads)), n, None, 1, None, None, 0, None)
    assert ("null resources" if fits else "too many rows") in say


@pytest.mark.parametrize("batch, beams, fits", [(2 ** 22 - 1, 1, True), (2 ** 22, 1, False), (2 ** 22 - 1, 4, True), (2 ** 21, 8, False),
                                                (2 ** 18 - 1, 64, True), (2 ** 18, 64, False)])
def test_beam_select_past_a_launch(batch, beams, fits):
    a = decoding._BeamStruct(vocab=100, batch=batch, beams=beams, keep=2, type=1)
    assert ("null resources" if fits else "too many rows") in _error("faiss_amd_beam_select", None, ctypes.byref(a), None)
    size = ctypes.c_size_t()
    assert ("null resources" if fits else "too many rows") in _error("faiss_amd_beam_select_workspace", None, ctypes.byref(a), ctypes.byref(size))


@pytest.mark.parametrize("batch, beams, keep, fits", [(2 ** 24 - 1, 1, 1, True), (2 ** 24, 1, 1, False), (2 ** 20, 100, 15, True), (2 ** 20, 100, 16, False)])
def test_reorder_beams_past_a_launch(batch, beams, keep, fits):
    say = _error("faiss_amd_reorder_beams", None, 1, None, None, batch, beams, keep, 0, None)
    assert ("null resources" if fits else "too many rows") in say


@pytest.mark.parametrize("batch, beams, fits", [(2 ** 24 - 1, 1, True), (2 ** 24, 1, False), (2 ** 21 - 1, 8, True), (2 ** 21, 8, False)])
def test_fork_blocks_past_a_launch(batch, beams, fits):
    a = decoding._ForkStruct(tableStride=4, batch=batch, beams=beams, numColumns=4)
    assert ("null resources" if fits else "too many rows") in _error("faiss_amd_fork_blocks", None, 1, ctypes.byref(_cache()), ctypes.byref(a), None)


@pytest.mark.parametrize("batch, heads, kv, fits", [(10 ** 6, 8, 2, True), (2 ** 22, 2, 2, True), (2 ** 23, 2, 2, False), (2 ** 24, 16, 1, False)])
def test_attend_past_a_launch(batch, heads, kv, fits):
    # a work item of 256 threads is (request, key-value head, 16 rows) here, and some more for contexts that are split
    a = decoding._AttendStruct(tableStride=40, batch=batch, tokens=batch, heads=heads, numColumns=40, maxQueries=1, type=3, causal=1, scale=0.125)
    say = _error("faiss_amd_PagedCache_attend", None, ctypes.byref(_cache(numHeads=kv)), ctypes.byref(a), None)
    assert ("null resources" if fits else "too many rows") in say


class _Res:  # what the wrappers look at before the library sees the call
    device = 0
    _h = None
    _lib = None


def _cache_on_the_host():
    c = decoding.PagedCache.__new__(decoding.PagedCache)
    c.res, c.num_heads, c.head_dim = _Res, 2, 64
    return c


def test_gradients_are_not_dropped():
    """no operator has a backward pass: a tensor that requires a gradient is refused, unless none is recorded"""
    i32 = torch.int32
    c, x, n = _cache_on_the_host(), torch.zeros((3, 2, 64), dtype=torch.float16), torch.zeros(3, dtype=i32)
    g = x.clone().requires_grad_()
    table, parents = torch.zeros((3, 4), dtype=i32), torch.zeros((1, 2), dtype=i32)
    logits, scores = torch.zeros((1, 2, 5)), torch.zeros((1, 2))
    calls = [(lambda: c.attend(g, table, n), True), (lambda: c.attend(x, table, n), False), (lambda: c.add(g, x, n), True),
             (lambda: decoding.beam_select(_Res, logits.clone().requires_grad_(), scores, 2), True),
             (lambda: decoding.beam_select(_Res, logits, scores, 2), False)]
    for call, refused in calls:
        with pytest.raises(ValueError, match="gradient" if refused else "device"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="device"):
            call()
        with torch.inference_mode(), pytest.raises(ValueError, match="device"):
            call()
    with pytest.raises(ValueError, match="device"):  # (looked at first)
        decoding.reorder_beams(_Res, [g], parents)


def test_lazily_negated_and_conjugated_tensors_are_refused():
    """their memory holds other numbers than the tensor does"""
    i32 = torch.int32
    c, n, table, parents = _cache_on_the_host(), torch.zeros(3, dtype=i32), torch.zeros((3, 4), dtype=i32), torch.zeros((1, 2), dtype=i32)
    z = torch.randn((1, 2, 5), dtype=torch.complex64)
    neg = z.conj().imag
    assert neg.is_neg()
    scores = torch.zeros((1, 2))
    for call in (lambda: decoding.beam_select(_Res, neg, scores, 2), lambda: decoding.beam_select(_Res, torch._neg_view(neg.clone()), scores, 2)):
        with pytest.raises(ValueError, match="lazily"):
            call()
    half = torch._neg_view(torch.zeros((3, 2, 64), dtype=torch.float16))
    for call in (lambda: c.attend(half, table, n), lambda: c.add(half, half, n)):
        with pytest.raises(ValueError, match="lazily"):
            call()


def test_what_is_no_tensor_is_a_type_error():
    t = torch.zeros((1, 1, 16, 64), dtype=torch.int8)
    s = torch.zeros((1, 1))
    for k, v in (([0], t), (t, [0]), (None, None)):
        with pytest.raises(TypeError):
            decoding.PagedCache.wrap(_Res, k, v, s, s)
    with pytest.raises(ValueError, match="device"):
        decoding.PagedCache.wrap(_Res, t, t, s, s)
