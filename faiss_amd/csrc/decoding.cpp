// faiss_amd/csrc/decoding.cpp -- checks of the decoding operators' arguments (include/faiss_amd_c.h says what each call takes).
#include "decoding.h"
#include <cmath>
#include <vector>
#include "../../include/faiss_amd_c.h"
#include "index.h"

namespace faiss_amd {
namespace {

// memory of the resources' device; checked: the caller has looked
void on_device(const GpuResources& r, const void* p, const char* what, int checked) {
    if (!p) FA_THROW_MSG(std::string(what) + " must be provided (passed null)");
    if (checked) return;
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
        (void)hipGetLastError();
        FA_THROW_MSG(std::string(what) + " is not device memory");
    }
    if (a.type != hipMemoryTypeManaged && (a.type != hipMemoryTypeDevice || a.device != r.device))
        FA_THROW_MSG(std::string(what) + " is not memory of the resources' device");
}
void aligned(const void* p, size_t n, const char* what) {
    if ((uintptr_t)p % n) FA_THROW_MSG(std::string(what) + " is not aligned to " + std::to_string(n) + " bytes");
}

// A launch holds less than 2^32 threads.  All of a call's launches are checked before the first one: it is refused as a whole
void launchable(int64_t workgroups, int threads, const char* call) {
    if (workgroups * threads >= (int64_t)1 << 32) FA_THROW_MSG(std::string(call) + ": too many rows for one call");
}

// the calling thread's device is the resources' one while a call checks its memory and launches its work
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(const GpuResources* r) {
        if (!r) FA_THROW_MSG("null resources handle");
        int now = 0;
        HIP_CHECK(hipGetDevice(&now));
        if (now == r->device) return;
        HIP_CHECK(hipSetDevice(r->device));
        before = now;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

CacheView view(const FaissAmdPagedCache* c) {
    FA_THROW_IF_NOT_MSG(c, "null cache");
    FA_THROW_IF_NOT_MSG(c->code == CACHE_INT8 || c->code == CACHE_E4M3, "cache code must be 0 (int8) or 1 (e4m3)");
    FA_THROW_IF_NOT_MSG(c->blockSize == 16 || c->blockSize == 32 || c->blockSize == 64 || c->blockSize == 128 || c->blockSize == 256,
                        "block size must be 16, 32, 64, 128 or 256");
    FA_THROW_IF_NOT_MSG(c->headDim == 64 || c->headDim == 96 || c->headDim == 128 || c->headDim == 192 || c->headDim == 256,
                        "head dimension must be 64, 96, 128, 192 or 256");
    FA_THROW_IF_NOT_MSG(c->numHeads >= 1 && c->numHeads <= 32767, "number of heads out of range");
    FA_THROW_IF_NOT_MSG(c->numBlocks >= 1 && (int64_t)c->numBlocks * c->blockSize < ((int64_t)1 << 31), "number of blocks out of range");
    // (the attention counts a block's place in units of 512 bytes)
    FA_THROW_IF_NOT_MSG((double)c->numBlocks * c->numHeads * c->blockSize * c->headDim < 2e12, "cache too large");
    CacheView v;
    v.k = (uint8_t*)c->keys;
    v.v = (uint8_t*)c->values;
    v.ks = c->keyScales;
    v.vs = c->valueScales;
    v.code = c->code;
    v.numBlocks = c->numBlocks;
    v.blockSize = c->blockSize;
    v.numHeads = c->numHeads;
    v.headDim = c->headDim;
    return v;
}
void check_memory(const GpuResources& r, const CacheView& v, int checked) {
    on_device(r, v.k, "cache keys", checked);
    on_device(r, v.v, "cache values", checked);
    on_device(r, v.ks, "cache keyScales", checked);
    on_device(r, v.vs, "cache valueScales", checked);
    aligned(v.k, 16, "cache keys");
    aligned(v.v, 16, "cache values");
    aligned(v.ks, 4, "cache keyScales");
    aligned(v.vs, 4, "cache valueScales");
}
bool half_type(int t) { return t == DT_F16 || t == DT_BF16; }
size_t type_size(int t) { return t == DT_F32 ? 4 : 2; }

} // namespace

void plan_blocks(const GpuResources* r, const FaissAmdPlanBlocksParams* p, hipStream_t stream) {
    FA_THROW_IF_NOT_MSG(p, "null arguments");
    FA_THROW_IF_NOT_MSG(p->batch >= 0 && p->numColumns >= 0 && p->maxTokens >= 0, "plan_blocks: negative size");
    FA_THROW_IF_NOT_MSG(p->batch <= 1 << 24, "plan_blocks: batch too large");
    FA_THROW_IF_NOT_MSG(p->blockSize >= 1 && p->numBlocks >= 1 && (int64_t)p->numBlocks * p->blockSize < ((int64_t)1 << 31),
                        "plan_blocks: number of blocks out of range");
    FA_THROW_IF_NOT_MSG((int64_t)p->numColumns * p->blockSize < ((int64_t)1 << 31), "plan_blocks: table too wide");
    FA_THROW_IF_NOT_MSG(p->tableStride >= p->numColumns && (!p->ownedTable || p->ownedStride >= p->numColumns), "plan_blocks: rows of the table overlap");
    launchable((int64_t)p->batch + (int64_t)div_up(p->maxTokens, kPlanSlots), 256, "plan_blocks");
    const int checked = p->pointersChecked;
    DeviceScope scope(r);
    if (p->batch > 0) {
        if (p->numColumns > 0) on_device(*r, p->blockTable, "blockTable", checked);
        if (p->ownedTable) on_device(*r, p->ownedTable, "ownedTable", checked);
        on_device(*r, p->lengths, "lengths", checked);
        on_device(*r, p->newLengths, "newLengths", checked);
        on_device(*r, p->lengthsOut, "lengthsOut", checked);
        on_device(*r, p->granted, "granted", checked);
    }
    on_device(*r, p->freeRing, "freeRing", checked);
    on_device(*r, p->freeState, "freeState", checked);
    on_device(*r, p->freeStateOut, "freeStateOut", checked);
    on_device(*r, p->queryOffsets, "queryOffsets", checked);
    on_device(*r, p->workspace, "workspace", checked);
    if (p->maxTokens > 0) on_device(*r, p->slots, "slots", checked);
    PlanArgs a;
    a.table = p->blockTable;
    a.owned = p->ownedTable;
    a.tableStride = p->tableStride;
    a.ownedStride = p->ownedStride;
    a.lengths = p->lengths;
    a.newLengths = p->newLengths;
    a.ring = p->freeRing;
    a.state = p->freeState;
    a.lengthsOut = p->lengthsOut;
    a.stateOut = p->freeStateOut;
    a.queryOffsets = p->queryOffsets;
    a.slots = p->slots;
    a.granted = p->granted;
    a.scratch = p->workspace;
    a.batch = p->batch;
    a.cols = p->numColumns;
    a.numBlocks = p->numBlocks;
    a.blockSize = p->blockSize;
    a.maxTokens = p->maxTokens;
    launch_plan_blocks(a, stream);
}

void cache_add(const GpuResources* r, const FaissAmdPagedCache* c, const FaissAmdCacheAddParams* p, hipStream_t stream) {
    AddArgs a;
    a.cache = view(c);
    FA_THROW_IF_NOT_MSG(p, "null arguments");
    FA_THROW_IF_NOT_MSG(half_type(p->type), "add: keys and values must be float16 or bfloat16");
    FA_THROW_IF_NOT_MSG(p->tokens >= 0 && p->tokens <= 1 << 30, "add: number of tokens out of range");
    const int checked = p->pointersChecked;
    DeviceScope scope(r);
    if (p->tokens == 0) return;
    check_memory(*r, a.cache, checked);
    on_device(*r, p->keys, "keys", checked);
    on_device(*r, p->values, "values", checked);
    on_device(*r, p->slots, "slots", checked);
    aligned(p->keys, 2, "keys");
    aligned(p->values, 2, "values");
    if (p->tokens > kAddScan) on_device(*r, p->workspace, "workspace", checked);
    a.key = p->keys;
    a.value = p->values;
    a.keyTokenStride = p->keyTokenStride;
    a.keyHeadStride = p->keyHeadStride;
    a.valueTokenStride = p->valueTokenStride;
    a.valueHeadStride = p->valueHeadStride;
    a.slots = p->slots;
    a.workspace = p->workspace;
    a.tokens = p->tokens;
    a.type = p->type;
    launch_cache_add(a, stream);
}

void cache_reconstruct(const GpuResources* r, const FaissAmdPagedCache* c, int n, const int* blocks, int type, void* keys, void* values, int checked, hipStream_t stream) {
    ReconstructArgs a;
    a.cache = view(c);
    FA_THROW_IF_NOT_MSG(type == DT_F32 || half_type(type), "reconstruct: type must be float32, float16 or bfloat16");
    FA_THROW_IF_NOT_MSG(n >= 0, "reconstruct: negative number of blocks");
    launchable((int64_t)n * c->numHeads, 256, "reconstruct");
    DeviceScope scope(r);
    if (n == 0) return;
    check_memory(*r, a.cache, checked);
    on_device(*r, blocks, "blocks", checked);
    on_device(*r, keys, "keys", checked);
    on_device(*r, values, "values", checked);
    aligned(keys, 16, "keys");
    aligned(values, 16, "values");
    a.blocks = blocks;
    a.key = keys;
    a.value = values;
    a.n = n;
    a.type = type;
    launch_cache_reconstruct(a, stream);
}

void cache_attend(const GpuResources* r, const FaissAmdPagedCache* c, const FaissAmdAttendParams* p, hipStream_t stream, size_t* bytes) {
    AttendArgs a;
    a.cache = view(c);
    FA_THROW_IF_NOT_MSG(p, "null arguments");
    FA_THROW_IF_NOT_MSG(half_type(p->type), "attend: queries must be float16 or bfloat16");
    FA_THROW_IF_NOT_MSG(p->batch >= 0 && p->tokens >= 0 && p->numColumns >= 0 && p->maxQueries >= 0, "attend: negative size");
    FA_THROW_IF_NOT_MSG(p->heads >= 1 && p->heads % c->numHeads == 0, "attend: heads must be a multiple of the cache's heads");
    FA_THROW_IF_NOT_MSG(p->heads <= 65535 && (int64_t)p->tokens * p->heads < ((int64_t)1 << 31), "attend: too many rows for one call");
    FA_THROW_IF_NOT_MSG(((int64_t)p->numColumns + 1) * c->blockSize < ((int64_t)1 << 31), "attend: table too wide");
    FA_THROW_IF_NOT_MSG(p->tableStride >= p->numColumns, "attend: rows of the table overlap");
    FA_THROW_IF_NOT_MSG(p->queryOffsets || p->tokens == p->batch, "attend: one query per request without queryOffsets");
    FA_THROW_IF_NOT_MSG(std::isfinite(p->scale), "attend: scale must be finite");
    a.q = p->queries;
    a.out = p->out;
    a.lse = p->lse;
    a.qTokenStride = p->queryTokenStride;
    a.qHeadStride = p->queryHeadStride;
    a.outTokenStride = p->outTokenStride;
    a.outHeadStride = p->outHeadStride;
    a.table = p->blockTable;
    a.tableStride = p->tableStride;
    a.lengths = p->lengths;
    a.queryOffsets = p->queryOffsets;
    a.batch = p->batch;
    a.tokens = p->tokens;
    a.heads = p->heads;
    a.cols = p->numColumns;
    a.maxQueries = p->queryOffsets ? std::min(std::max(p->maxQueries, 1), std::max(p->tokens, 1)) : 1;
    a.type = p->type;
    a.causal = p->causal ? 1 : 0;
    a.scale = p->scale;
    a.workspace = p->workspace;
    a.workspaceBytes = p->workspaceBytes;
    launchable(cache_attend_threads(a), 1, "attend");
    const int checked = p->pointersChecked;
    DeviceScope scope(r);
    const size_t need = cache_attend_workspace(a, r->num_cus);
    if (bytes) {
        *bytes = need;
        return;
    }
    if (p->batch == 0 || p->tokens == 0) return;
    check_memory(*r, a.cache, checked);
    on_device(*r, p->queries, "queries", checked);
    on_device(*r, p->out, "out", checked);
    aligned(p->queries, 2, "queries");
    aligned(p->out, 2, "out");
    if (p->lse) on_device(*r, p->lse, "lse", checked);
    if (p->numColumns > 0) on_device(*r, p->blockTable, "blockTable", checked);
    on_device(*r, p->lengths, "lengths", checked);
    if (p->queryOffsets) on_device(*r, p->queryOffsets, "queryOffsets", checked);
    if (need) {
        FA_THROW_IF_NOT_MSG(p->workspaceBytes >= need, "attend: workspace too small");
        on_device(*r, p->workspace, "workspace", checked);
        aligned(p->workspace, 256, "workspace");
    }
    launch_cache_attend(a, r->num_cus, stream);
}

void beam_select(const GpuResources* r, const FaissAmdBeamSelectParams* p, hipStream_t stream, size_t* bytes) {
    FA_THROW_IF_NOT_MSG(p, "null arguments");
    FA_THROW_IF_NOT_MSG(p->type == DT_F32 || half_type(p->type), "beam_select: logits must be float32, float16 or bfloat16");
    FA_THROW_IF_NOT_MSG(p->batch >= 0, "beam_select: negative batch");
    FA_THROW_IF_NOT_MSG(p->beams >= 1 && p->beams <= kMaxBeams && p->keep >= 1 && p->keep <= kMaxBeams, "beam_select: beams and beams kept must be in [1, 64]");
    launchable((int64_t)p->batch * p->beams, 256, "beam_select"); // (rows are split while there are few)
    launchable(p->batch, kBeamJoin, "beam_select");
    FA_THROW_IF_NOT_MSG(p->vocab >= 1 && p->vocab < ((int64_t)1 << 31), "beam_select: vocabulary out of range");
    FA_THROW_IF_NOT_MSG(p->padToken >= 0 && p->padToken < p->vocab, "beam_select: padToken is no token");
    BeamArgs a;
    a.logits = p->logits;
    a.batchStride = p->batchStride;
    a.beamStride = p->beamStride;
    a.scores = p->scores;
    a.finished = p->finished;
    a.outScores = p->outScores;
    a.parents = p->outParents;
    a.tokens = p->outTokens;
    a.vocab = p->vocab;
    a.batch = p->batch;
    a.beams = p->beams;
    a.keep = p->keep;
    a.padToken = p->padToken;
    a.type = p->type;
    a.workspace = p->workspace;
    a.workspaceBytes = p->workspaceBytes;
    const int checked = p->pointersChecked;
    DeviceScope scope(r);
    const size_t need = beam_select_workspace(a, r->num_cus);
    if (bytes) {
        *bytes = need;
        return;
    }
    if (p->batch == 0) return;
    on_device(*r, p->logits, "logits", checked);
    aligned(p->logits, type_size(p->type), "logits");
    on_device(*r, p->scores, "scores", checked);
    if (p->finished) on_device(*r, p->finished, "finished", checked);
    on_device(*r, p->outScores, "outScores", checked);
    on_device(*r, p->outParents, "outParents", checked);
    on_device(*r, p->outTokens, "outTokens", checked);
    FA_THROW_IF_NOT_MSG(p->workspaceBytes >= need, "beam_select: workspace too small");
    on_device(*r, p->workspace, "workspace", checked);
    aligned(p->workspace, 256, "workspace");
    launch_beam_select(a, r->num_cus, stream);
}

void reorder_beams(const GpuResources* r, int n, const FaissAmdBeamState* states, const int* parents, int batch, int beams, int keep, int checked, hipStream_t stream) {
    FA_THROW_IF_NOT_MSG(n >= 0 && batch >= 0 && beams >= 1 && keep >= 0, "reorder_beams: negative size");
    FA_THROW_IF_NOT_MSG((int64_t)batch * keep < ((int64_t)1 << 31) && (int64_t)batch * beams < ((int64_t)1 << 31), "reorder_beams: too many rows");
    launchable((int64_t)batch * keep, 256, "reorder_beams");
    DeviceScope scope(r);
    if (n == 0 || batch == 0 || keep == 0) return;
    FA_THROW_IF_NOT_MSG(states, "reorder_beams: null states");
    on_device(*r, parents, "parents", checked);
    std::vector<ReorderState> st((size_t)n);
    for (int i = 0; i < n; ++i) {
        const FaissAmdBeamState& s = states[i];
        FA_THROW_IF_NOT_MSG(s.rowBytes >= 0 && s.batchBytes >= 0 && s.beamBytes >= 0, "reorder_beams: negative stride");
        st[i] = {s.in, s.out, s.batchBytes, s.beamBytes, s.rowBytes};
        if (s.rowBytes == 0) continue;
        on_device(*r, s.in, "a state's input", checked);
        on_device(*r, s.out, "a state's output", checked);
        const uintptr_t i0 = (uintptr_t)s.in, i1 = i0 + (uintptr_t)((batch - 1) * s.batchBytes + (beams - 1) * s.beamBytes + s.rowBytes);
        const uintptr_t o0 = (uintptr_t)s.out, o1 = o0 + (uintptr_t)((int64_t)batch * keep * s.rowBytes);
        FA_THROW_IF_NOT_MSG(o1 <= i0 || i1 <= o0, "reorder_beams: a state's output overlaps its input");
    }
    launch_beam_reorder(st.data(), n, parents, batch, beams, keep, stream);
}

void fork_blocks(const GpuResources* r, int n, const FaissAmdPagedCache* caches, const FaissAmdForkBlocksParams* p, hipStream_t stream) {
    FA_THROW_IF_NOT_MSG(p, "null arguments");
    FA_THROW_IF_NOT_MSG(n >= 1 && caches, "fork_blocks: at least one cache");
    FA_THROW_IF_NOT_MSG(p->batch >= 0 && p->beams >= 1 && p->numColumns >= 0, "fork_blocks: negative size");
    FA_THROW_IF_NOT_MSG((int64_t)p->batch * p->beams < ((int64_t)1 << 31), "fork_blocks: too many rows");
    launchable((int64_t)p->batch * p->beams, 256, "fork_blocks");
    FA_THROW_IF_NOT_MSG(p->tableStride >= p->numColumns && (!p->ownedTable || p->ownedStride >= p->numColumns), "fork_blocks: rows of the table overlap");
    std::vector<CacheView> v((size_t)n);
    for (int i = 0; i < n; ++i) {
        v[i] = view(&caches[i]);
        FA_THROW_IF_NOT_MSG(v[i].blockSize == v[0].blockSize && v[i].numBlocks == v[0].numBlocks, "fork_blocks: caches of different blocks");
    }
    FA_THROW_IF_NOT_MSG((int64_t)p->numColumns * v[0].blockSize < ((int64_t)1 << 31), "fork_blocks: table too wide");
    const int checked = p->pointersChecked;
    DeviceScope scope(r);
    if (p->batch == 0) return;
    for (int i = 0; i < n; ++i) check_memory(*r, v[i], checked);
    if (p->numColumns > 0) {
        on_device(*r, p->blockTable, "blockTable", checked);
        on_device(*r, p->tableOut, "tableOut", checked);
        FA_THROW_IF_NOT_MSG(p->tableOut != p->blockTable && p->ownedTable != p->blockTable && (!p->ownedTable || p->ownedTable != p->tableOut),
                            "fork_blocks: outputs overlap inputs");
        if (p->ownedTable) on_device(*r, p->ownedTable, "ownedTable", checked);
    }
    on_device(*r, p->lengths, "lengths", checked);
    on_device(*r, p->spare, "spare", checked);
    on_device(*r, p->parents, "parents", checked);
    on_device(*r, p->lengthsOut, "lengthsOut", checked);
    on_device(*r, p->spareOut, "spareOut", checked);
    FA_THROW_IF_NOT_MSG(p->lengthsOut != p->lengths && p->spareOut != p->spare, "fork_blocks: outputs overlap inputs");
    ForkArgs a;
    a.table = p->blockTable;
    a.tableStride = p->tableStride;
    a.lengths = p->lengths;
    a.spare = p->spare;
    a.parents = p->parents;
    a.tableOut = p->tableOut;
    a.lengthsOut = p->lengthsOut;
    a.spareOut = p->spareOut;
    a.owned = p->ownedTable;
    a.ownedStride = p->ownedStride;
    a.batch = p->batch;
    a.beams = p->beams;
    a.cols = p->numColumns;
    launch_fork_blocks(a, v.data(), n, stream);
}

} // namespace faiss_amd
