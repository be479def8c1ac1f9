"""faiss_amd/decoding.py -- operators of a program that decodes with a model next to its searches, over torch tensors.

    cache = PagedCache(res, num_blocks, block_size, num_heads, head_dim, code="e4m3")   # one per layer
    plan = plan_blocks(res, table, lengths, new_lengths, ring, state, block_size, max_tokens, owned_table=owned)
    cache.add(k, v, plan.slots)
    out = cache.attend(q, table, plan.lengths, query_offsets=plan.query_offsets)
    scores, parents, tokens = beam_select(res, logits, scores, num_beams)
    states = reorder_beams(res, states, parents)
    table, lengths, spare = fork_blocks(res, caches, table, lengths, spare, parents, owned_table=owned)

The work of a call is ordered on torch's current stream of the resources' device and nothing is synchronised, so calls can be
captured into a graph; results and scratch come from torch's allocator.  What the calls compute, and what they do with lengths,
slots, block ids and parents that are out of range, is stated in include/faiss_amd_c.h.  Tensors must be on the resources'
device; arguments of the wrong shape, type or device raise ValueError / TypeError before anything is launched.  Nothing here has a
backward pass: a tensor that requires a gradient is refused while gradients are recorded (torch.no_grad() says that none is meant).
"""
import collections
import ctypes
import math

import torch

from . import _check, load_library

_HALF = {torch.float16: 2, torch.bfloat16: 3}
_FLOAT = {torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
_CODES = {"int8": 0, "e4m3": 1}
_CODE_OF = {torch.int8: 0, torch.float8_e4m3fn: 1}
_P, _I, _I64, _F, _SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class _CacheStruct(ctypes.Structure):
    _fields_ = [("keys", _P), ("values", _P), ("keyScales", _P), ("valueScales", _P), ("code", _I), ("numBlocks", _I),
                ("blockSize", _I), ("numHeads", _I), ("headDim", _I)]


class _PlanStruct(ctypes.Structure):
    _fields_ = [("blockTable", _P), ("ownedTable", _P), ("tableStride", _I64), ("ownedStride", _I64), ("lengths", _P),
                ("newLengths", _P), ("freeRing", _P), ("freeState", _P), ("lengthsOut", _P), ("freeStateOut", _P),
                ("queryOffsets", _P), ("slots", _P), ("granted", _P), ("workspace", _P), ("batch", _I), ("numColumns", _I),
                ("numBlocks", _I), ("blockSize", _I), ("maxTokens", _I), ("pointersChecked", _I)]


class _AddStruct(ctypes.Structure):
    _fields_ = [("keys", _P), ("values", _P), ("keyTokenStride", _I64), ("keyHeadStride", _I64), ("valueTokenStride", _I64),
                ("valueHeadStride", _I64), ("slots", _P), ("tokens", _I), ("type", _I), ("pointersChecked", _I),
                ("workspace", _P)]


class _AttendStruct(ctypes.Structure):
    _fields_ = [("queries", _P), ("out", _P), ("lse", _P), ("queryTokenStride", _I64), ("queryHeadStride", _I64),
                ("outTokenStride", _I64), ("outHeadStride", _I64), ("blockTable", _P), ("tableStride", _I64), ("lengths", _P),
                ("queryOffsets", _P), ("batch", _I), ("tokens", _I), ("heads", _I), ("numColumns", _I), ("maxQueries", _I),
                ("type", _I), ("causal", _I), ("pointersChecked", _I), ("scale", _F), ("workspace", _P), ("workspaceBytes", _SZ)]


class _BeamStruct(ctypes.Structure):
    _fields_ = [("logits", _P), ("batchStride", _I64), ("beamStride", _I64), ("scores", _P), ("finished", _P), ("outScores", _P),
                ("outParents", _P), ("outTokens", _P), ("vocab", _I64), ("batch", _I), ("beams", _I), ("keep", _I),
                ("padToken", _I), ("type", _I), ("pointersChecked", _I), ("workspace", _P), ("workspaceBytes", _SZ)]


class _StateStruct(ctypes.Structure):
    _fields_ = [("in_", _P), ("out", _P), ("batchBytes", _I64), ("beamBytes", _I64), ("rowBytes", _I64)]


class _ForkStruct(ctypes.Structure):
    _fields_ = [("blockTable", _P), ("tableStride", _I64), ("lengths", _P), ("spare", _P), ("parents", _P), ("tableOut", _P),
                ("lengthsOut", _P), ("spareOut", _P), ("batch", _I), ("beams", _I), ("numColumns", _I), ("pointersChecked", _I),
                ("ownedTable", _P), ("ownedStride", _I64)]


_byref = ctypes.byref


def _tensor(res, t, name, dtype=None, dim=None, dense=True):
    """`t` is a tensor of res's device with the dtype(s), number of dimensions and (dense) the contiguous layout asked for"""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if dim is not None and t.dim() != dim:
        raise ValueError("%s must have %d dimensions, not %d" % (name, dim, t.dim()))
    if dtype is not torch.int32:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("%s requires a gradient, which this call does not give" % name)
        if t.is_neg() or t.is_conj():  # (the memory holds other numbers than the tensor)
            raise ValueError("%s is negated or conjugated lazily: resolve_neg() or resolve_conj() first" % name)
    if not t.is_cuda or t.device.index != res.device:
        raise ValueError("%s must be on the resources' device cuda:%d, not %s" % (name, res.device, t.device))
    if dense and not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t


def _rows(res, t, name, dtype=torch.int32):
    """a table whose rows are dense and do not overlap"""
    _tensor(res, t, name, dtype, 2, dense=False)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("the rows of %s must be dense" % name)
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("the rows of %s must not overlap" % name)
    return t


def _row_stride(t):
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _same_length(t, n, name):
    if t.shape[0] != n:
        raise ValueError("%s must have %d entries, not %d" % (name, n, t.shape[0]))
    return t


def _dense_last(t, name):
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError("the last dimension of %s must be dense" % name)


def _rows_apart(t, name):
    """no two rows of t [n, m, dense] share memory (or are interleaved): one of two results would stand there"""
    reach = t.shape[2]
    for stride, n in sorted((t.stride(i), t.shape[i]) for i in (0, 1)):
        if n > 1 and stride < reach:
            raise ValueError("the rows of %s must not overlap" % name)
        reach += stride * (n - 1) if n > 1 else 0


try:  # the same number without a Stream object around it (a microsecond of every call)
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # a torch without CUDA / HIP

    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream


def _stream(res):
    return _raw_stream(res.device)


def _device(res):
    return torch.device("cuda", res.device)


BlockPlan = collections.namedtuple("BlockPlan", "lengths free_state query_offsets slots granted")


def plan_blocks(res, block_table, lengths, new_lengths, free_ring, free_state, block_size, max_tokens, owned_table=None,
                lengths_out=None, free_state_out=None):
    """Block tables and slot maps on the device from request lengths (faiss_amd_plan_blocks).

    block_table [batch, columns] and free_ring [num_blocks] (int32) are updated in place; lengths, new_lengths [batch] int32;
    free_state [2] int64 = {front, count}; lengths_out / free_state_out may be the tensors given (None: new ones).  ->
    BlockPlan(lengths [batch], free_state, query_offsets [batch + 1], slots [max_tokens], granted [batch])."""
    _rows(res, block_table, "block_table")
    n, cols = block_table.shape
    for t, name in ((lengths, "lengths"), (new_lengths, "new_lengths")):
        _same_length(_tensor(res, t, name, torch.int32, 1), n, name)
    _tensor(res, free_ring, "free_ring", torch.int32, 1)
    _same_length(_tensor(res, free_state, "free_state", torch.int64, 1), 2, "free_state")
    if owned_table is not None:
        _rows(res, owned_table, "owned_table")
        if owned_table.shape != block_table.shape:
            raise ValueError("owned_table must have the shape of block_table")
    dev = _device(res)
    if lengths_out is not None:
        _same_length(_tensor(res, lengths_out, "lengths_out", torch.int32, 1), n, "lengths_out")
    if free_state_out is None:
        free_state_out = torch.empty(2, dtype=torch.int64, device=dev)
    else:
        _same_length(_tensor(res, free_state_out, "free_state_out", torch.int64, 1), 2, "free_state_out")
    max_tokens, block_size = int(max_tokens), int(block_size)
    if not (0 <= max_tokens < 1 << 31 and 1 <= block_size < 1 << 31):
        raise ValueError("block_size or max_tokens out of range")
    # everything that is made here in one allocation
    made = 0 if lengths_out is not None else n
    offsets, granted, scratch, slots, own = torch.empty(6 * n + 3 + max_tokens + made, dtype=torch.int32, device=dev).split(
        [n + 1, n, 4 * n + 2, max_tokens, made])
    if lengths_out is None:
        lengths_out = own
    a = _PlanStruct(block_table.data_ptr() or None, owned_table.data_ptr() if owned_table is not None else None,
                    _row_stride(block_table), _row_stride(owned_table) if owned_table is not None else 0, lengths.data_ptr() or None,
                    new_lengths.data_ptr() or None, free_ring.data_ptr() or None, free_state.data_ptr(), lengths_out.data_ptr() or None,
                    free_state_out.data_ptr(), offsets.data_ptr(), slots.data_ptr() or None, granted.data_ptr(), scratch.data_ptr(),
                    n, cols, free_ring.shape[0], block_size, max_tokens, 1)
    _check(res._lib.faiss_amd_plan_blocks(res._h, _byref(a), _stream(res)))
    return BlockPlan(lengths_out, free_state_out, offsets, slots, granted)


class PagedCache:
    """Keys and values of one layer in blocks of 8-bit codes, one scale per block and head.

    Tensors: k_codes [num_blocks, num_heads, block_size, head_dim], v_codes [num_blocks, num_heads, head_dim, block_size]
    (torch.int8 or torch.float8_e4m3fn), k_scales, v_scales [num_blocks, num_heads] float32; a value is code * scale."""

    def __init__(self, res, num_blocks, block_size, num_heads, head_dim, code="e4m3"):
        if code not in _CODES:
            raise ValueError("code must be 'int8' or 'e4m3'")
        dt = torch.int8 if code == "int8" else torch.float8_e4m3fn
        dev = _device(res)
        k = torch.zeros((num_blocks, num_heads, block_size, head_dim), dtype=torch.int8, device=dev).view(dt)
        v = torch.zeros((num_blocks, num_heads, head_dim, block_size), dtype=torch.int8, device=dev).view(dt)
        self._set(res, k, v, torch.zeros((num_blocks, num_heads), device=dev), torch.zeros((num_blocks, num_heads), device=dev))

    @classmethod
    def wrap(cls, res, k_codes, v_codes, k_scales, v_scales):
        """a cache over tensors that the caller holds"""
        self = cls.__new__(cls)
        self._set(res, k_codes, v_codes, k_scales, v_scales)
        return self

    def _set(self, res, k, v, ks, vs):
        if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
            raise TypeError("codes must be torch tensors")
        if k.dtype not in _CODE_OF or v.dtype != k.dtype:
            raise TypeError("codes must be torch.int8 or torch.float8_e4m3fn, keys and values alike")
        _tensor(res, k, "k_codes", None, 4)
        _tensor(res, v, "v_codes", None, 4)
        n, h, b, d = k.shape
        if tuple(v.shape) != (n, h, d, b):
            raise ValueError("v_codes must have the shape %s, not %s" % ((n, h, d, b), tuple(v.shape)))
        for t, name in ((ks, "k_scales"), (vs, "v_scales")):
            if tuple(_tensor(res, t, name, torch.float32, 2).shape) != (n, h):
                raise ValueError("%s must have the shape %s" % (name, (n, h)))
        if b not in (16, 32, 64, 128, 256):
            raise ValueError("block size must be 16, 32, 64, 128 or 256")
        if d not in (64, 96, 128, 192, 256):
            raise ValueError("head dimension must be 64, 96, 128, 192 or 256")
        if n < 1 or h < 1 or n * b >= 1 << 31:
            raise ValueError("number of blocks or heads out of range")
        self.res, self.k_codes, self.v_codes, self.k_scales, self.v_scales = res, k, v, ks, vs
        self.num_blocks, self.num_heads, self.block_size, self.head_dim = n, h, b, d
        self.code = "int8" if k.dtype == torch.int8 else "e4m3"
        self._s = _CacheStruct(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), _CODE_OF[k.dtype], n, b, h, d)
        self._ref = _byref(self._s)
        self._lib = load_library()
        self._workspaces = {}

    def add(self, k, v, slots):
        """store the tokens k, v [tokens, num_heads, head_dim] (float16 / bfloat16) at slots [tokens] (int32; -1: skipped)"""
        res = self.res
        for t, name in ((k, "k"), (v, "v")):
            _tensor(res, t, name, None, 3, dense=False)
            if t.shape[1] != self.num_heads or t.shape[2] != self.head_dim:
                raise ValueError("%s must be [tokens, %d, %d]" % (name, self.num_heads, self.head_dim))
            _dense_last(t, name)
        if k.dtype not in _HALF or v.dtype != k.dtype:
            raise TypeError("k and v must be float16 or bfloat16, both the same")
        n = k.shape[0]
        _same_length(v, n, "v")
        _same_length(_tensor(res, slots, "slots", torch.int32, 1), n, "slots")
        a = _AddStruct(k.data_ptr() or None, v.data_ptr() or None, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                       slots.data_ptr() or None, n, _HALF[k.dtype], 1, None)
        if n > 512:  # (its blocks are listed)
            ws = torch.empty(3 * self.num_blocks + 1, dtype=torch.int32, device=k.device)
            a.workspace = ws.data_ptr()
        _check(self._lib.faiss_amd_PagedCache_add(res._h, self._ref, _byref(a), _stream(res)))

    def reconstruct(self, blocks, dtype=torch.float32):
        """the values of blocks [n] (int32) -> k, v [n, num_heads, block_size, head_dim]; NaN for an id out of range"""
        res = self.res
        _tensor(res, blocks, "blocks", torch.int32, 1)
        if dtype not in _FLOAT:
            raise TypeError("dtype must be float32, float16 or bfloat16")
        shape = (blocks.shape[0], self.num_heads, self.block_size, self.head_dim)
        k, v = torch.empty(shape, dtype=dtype, device=blocks.device), torch.empty(shape, dtype=dtype, device=blocks.device)
        _check(self._lib.faiss_amd_PagedCache_reconstruct(res._h, self._ref, shape[0], blocks.data_ptr() or None, _FLOAT[dtype],
                                                          k.data_ptr() or None, v.data_ptr() or None, 1, _stream(res)))
        return k, v

    def attend(self, q, block_table, lengths, query_offsets=None, scale=None, causal=True, max_queries=None, out=None,
               return_lse=False):
        """Attention of q [tokens, heads, head_dim] (float16 / bfloat16) over the cache -> out (, lse [tokens, heads]).

        block_table [batch, columns], lengths [batch] (int32): each request's blocks and tokens, its new ones included; request
        b's queries are the rows query_offsets[b] ... query_offsets[b + 1] - 1 (int32 [batch + 1]; None: row b) and stand at
        its end.  scale: 1 / sqrt(head_dim) by default.  max_queries: an upper bound of a request's queries, which saves
        work that only longer ones need.  Rows of no request are left as they are in `out` (zero if it is None);
        out may be q itself, and shares no other memory with it."""
        res = self.res
        _tensor(res, q, "q", None, 3, dense=False)
        if q.dtype not in _HALF:
            raise TypeError("q must be float16 or bfloat16")
        t, h, d = q.shape
        if d != self.head_dim or h < 1 or h % self.num_heads:
            raise ValueError("q must be [tokens, a multiple of %d, %d]" % (self.num_heads, self.head_dim))
        _dense_last(q, "q")
        _rows(res, block_table, "block_table")
        n = block_table.shape[0]
        _same_length(_tensor(res, lengths, "lengths", torch.int32, 1), n, "lengths")
        if query_offsets is None:
            if t != n:
                raise ValueError("without query_offsets q must have one row per request")
            most = 1
        else:
            _same_length(_tensor(res, query_offsets, "query_offsets", torch.int32, 1), n + 1, "query_offsets")
            most = t if max_queries is None else min(int(max_queries), t)
        if out is None:
            out = torch.empty((t, h, d), dtype=q.dtype, device=q.device) if query_offsets is None else torch.zeros(
                (t, h, d), dtype=q.dtype, device=q.device)
        else:
            _tensor(res, out, "out", q.dtype, 3, dense=False)
            if out.shape != q.shape:
                raise ValueError("out must have the shape of q")
            _dense_last(out, "out")
            _rows_apart(out, "out")
        lse = None
        if return_lse:
            lse = torch.full((t, h), -math.inf, device=q.device)
        a = _AttendStruct(q.data_ptr() or None, out.data_ptr() or None, lse.data_ptr() if return_lse else None, q.stride(0), q.stride(1),
                          out.stride(0), out.stride(1), block_table.data_ptr() or None, _row_stride(block_table), lengths.data_ptr() or None,
                          query_offsets.data_ptr() if query_offsets is not None else None, n, t, h, block_table.shape[1],
                          max(most, 0), _HALF[q.dtype], 1 if causal else 0, 1, 1.0 / math.sqrt(d) if scale is None else float(scale),
                          None, 0)
        lib, ref = self._lib, _byref(a)
        # (the size follows from these numbers alone)
        sizes = (n, t, h, block_table.shape[1], a.maxQueries, query_offsets is None)
        need = self._workspaces.get(sizes)
        if need is None:
            size = _SZ(0)
            _check(lib.faiss_amd_PagedCache_attend_workspace(res._h, self._ref, ref, _byref(size)))
            if len(self._workspaces) > 1000:
                self._workspaces.clear()
            need = self._workspaces[sizes] = size.value
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspaceBytes = ws.data_ptr(), need
        _check(lib.faiss_amd_PagedCache_attend(res._h, self._ref, ref, _stream(res)))
        return (out, lse) if return_lse else out


def beam_select(res, logits, scores, num_beams, finished=None, pad_token=0):
    """The num_beams best of each batch item's candidates beam x token -> (scores float32, parents int32, tokens int32), each
    [batch, num_beams], best first, ties to the lowest beam, then the lowest token (faiss_amd_beam_select).

    logits [batch, beams, vocab] (float32 / float16 / bfloat16), scores [batch, beams] float32; finished [batch, beams] (bool):
    such a beam's only candidate is pad_token with its score unchanged.  Fewer candidates: score -inf, parent and token -1."""
    _tensor(res, logits, "logits", None, 3, dense=False)
    if logits.dtype not in _FLOAT:
        raise TypeError("logits must be float32, float16 or bfloat16")
    n, w, v = logits.shape
    _dense_last(logits, "logits")
    if tuple(_tensor(res, scores, "scores", torch.float32, 2).shape) != (n, w):
        raise ValueError("scores must have the shape %s" % ((n, w),))
    if finished is not None:
        if tuple(_tensor(res, finished, "finished", None, 2).shape) != (n, w):
            raise ValueError("finished must have the shape %s" % ((n, w),))
        if finished.dtype not in (torch.bool, torch.uint8):
            raise TypeError("finished must be bool or uint8")
    k = int(num_beams)
    dev = logits.device
    if not 1 <= k <= 64:
        raise ValueError("num_beams must be in [1, 64]")
    if not 0 <= int(pad_token) < max(v, 1):
        raise ValueError("pad_token is no token of the vocabulary")
    out = torch.empty((n, k), device=dev)
    which = torch.empty((2, n, k), dtype=torch.int32, device=dev)
    parents, tokens = which[0], which[1]
    a = _BeamStruct(logits.data_ptr() or None, logits.stride(0), logits.stride(1), scores.data_ptr() or None,
                    finished.data_ptr() if finished is not None else None, out.data_ptr() or None, parents.data_ptr() or None,
                    tokens.data_ptr() or None, v, n, w, k, int(pad_token), _FLOAT[logits.dtype], 1, None, 0)
    lib, ref = res._lib, _byref(a)
    # (the size follows from these numbers alone)
    known = res.__dict__.setdefault("_beam_workspaces", {})
    need = known.get((n, w, v, k))
    if need is None:
        size = _SZ(0)
        _check(lib.faiss_amd_beam_select_workspace(res._h, ref, _byref(size)))
        if len(known) > 1000:
            known.clear()
        need = known[n, w, v, k] = size.value
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    a.workspace, a.workspaceBytes = ws.data_ptr() or None, need
    _check(lib.faiss_amd_beam_select(res._h, ref, _stream(res)))
    return out, parents, tokens


def reorder_beams(res, states, parents):
    """states: tensors [batch, beams, ...] of any type -> new tensors [batch, num, ...] with out[b, j] = state[b, parents[b, j]]
    (parents [batch, num] int32; a row whose parent is out of range becomes zero).  A state's rows must be dense."""
    _tensor(res, parents, "parents", torch.int32, 2)
    n, k = parents.shape
    outs, flat, w = [], [], None
    for i, t in enumerate(states):
        _tensor(res, t, "a state", dense=False)
        shape = t.shape
        if len(shape) < 2 or shape[0] != n:
            raise ValueError("states[%d] must be [%d, beams, ...]" % (i, n))
        if w is None:
            w = shape[1]
        if shape[1] != w or w < 1:
            raise ValueError("the states must have the same number of beams")
        row = shape[2:]
        size = t.element_size()
        width = math.prod(row) * size
        if t.is_contiguous():
            batch, beam = w * width, width
        else:
            dense = 1
            for m, st in zip(reversed(row), reversed(t.stride()[2:])):
                if m > 1 and st != dense and t.numel():
                    raise ValueError("the rows of states[%d] must be dense" % i)
                dense *= m
            batch, beam = t.stride(0) * size, t.stride(1) * size
        out = t.new_empty((n, k) + row)
        outs.append(out)
        flat += (t.data_ptr(), out.data_ptr(), batch, beam, width)
    if outs:
        # (the array of FaissAmdBeamState as what it is, five 64-bit numbers each)
        arr = (_I64 * len(flat))(*flat)
        _check(res._lib.faiss_amd_reorder_beams(res._h, len(outs), arr, parents.data_ptr() or None, n, w, k, 1, _stream(res)))
    return outs


def fork_blocks(res, caches, block_table, lengths, spare, parents, owned_table=None):
    """Reorders beams over paged caches (all the layers that block_table leads to): row b * beams + j takes over the blocks of row
    b * beams + parents[b, j]; full blocks are shared, a partly filled last one is copied into the row's spare block.  ->
    new (block_table, lengths, spare).  block_table [batch * beams, columns], lengths, spare [batch * beams], parents [batch,
    beams], all int32 (faiss_amd_fork_blocks).  owned_table (the shape of block_table, updated in place): the one given to
    plan_blocks for these rows; with it every block stays in one of owned_table, spare and the free blocks.  Without it the new
    spare blocks are still noted there: once the rows are released, take the spare blocks first given again.  The beams of an item
    shrink together, in one call of plan_blocks, to zero or to whole blocks."""
    _rows(res, block_table, "block_table")
    _tensor(res, parents, "parents", torch.int32, 2)
    n, w = parents.shape
    rows, cols = block_table.shape
    if rows != n * w:
        raise ValueError("block_table must have batch * beams = %d rows" % (n * w))
    for t, name in ((lengths, "lengths"), (spare, "spare")):
        _same_length(_tensor(res, t, name, torch.int32, 1), rows, name)
    if owned_table is not None:
        _rows(res, owned_table, "owned_table")
        if owned_table.shape != block_table.shape:
            raise ValueError("owned_table must have the shape of block_table")
    caches = list(caches)
    if not caches:
        raise ValueError("at least one cache")
    for c in caches:
        if not isinstance(c, PagedCache):
            raise TypeError("caches must be PagedCache objects")
        if c.res.device != res.device:
            raise ValueError("the caches must be on the resources' device")
    dev = block_table.device
    table, lens, sp = (torch.empty((rows, cols), dtype=torch.int32, device=dev), torch.empty(rows, dtype=torch.int32, device=dev),
                       torch.empty(rows, dtype=torch.int32, device=dev))
    arr = (_CacheStruct * len(caches))(*[c._s for c in caches])
    a = _ForkStruct(block_table.data_ptr() or None, _row_stride(block_table), lengths.data_ptr() or None, spare.data_ptr() or None,
                    parents.data_ptr() or None, table.data_ptr() or None, lens.data_ptr() or None, sp.data_ptr() or None, n, w, cols, 1,
                    owned_table.data_ptr() or None if owned_table is not None else None, _row_stride(owned_table) if owned_table is not None else 0)
    if rows:
        _check(res._lib.faiss_amd_fork_blocks(res._h, len(caches), arr, _byref(a), _stream(res)))
    return table, lens, sp
