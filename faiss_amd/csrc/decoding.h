// faiss_amd/csrc/decoding.h -- operators of a program that decodes with a model over an 8-bit paged cache of keys and values:
// block tables and slot maps, adding and reading back tokens, attention, beam selection and reordering.
//
// The cache of one layer: keys    [numBlocks][numHeads][blockSize][headDim] one byte each,
//                         values  [numBlocks][numHeads][headDim][blockSize] one byte each (a dimension's tokens are adjacent:
//                                 the second product of the attention reads them as matrix operands without a transpose),
//                         scales  [numBlocks][numHeads] fp32 for keys and for values; a value is code * scale.
// Every call is ordered on the stream it is given, keeps nothing behind and allocates nothing (scratch is the caller's).
#pragma once
#include "common.h"

namespace faiss_amd {

enum CacheCode : int { CACHE_INT8 = 0, CACHE_E4M3 = 1 };
enum DecodeType : int { DT_F32 = 1, DT_F16 = 2, DT_BF16 = 3 }; // the values of faiss::gpu::DistanceDataType

struct CacheView {
    uint8_t* k = nullptr;
    uint8_t* v = nullptr;
    float* ks = nullptr;
    float* vs = nullptr;
    int code = CACHE_INT8, numBlocks = 0, blockSize = 0, numHeads = 0, headDim = 0;
};

struct PlanArgs {
    int* table = nullptr; // [batch][tableStride], `cols` entries used
    int* owned = nullptr; // nullable: a second table that new blocks are noted in too and released blocks are read from
    int64_t tableStride = 0, ownedStride = 0;
    const int* lengths = nullptr;
    const int* newLengths = nullptr;
    int* ring = nullptr;
    const int64_t* state = nullptr; // {front, count}
    int* lengthsOut = nullptr;
    int64_t* stateOut = nullptr;
    int* queryOffsets = nullptr; // [batch + 1]
    int* slots = nullptr;        // [maxTokens]
    int* granted = nullptr;      // [batch]
    int* scratch = nullptr;      // plan_scratch_ints(batch) ints
    int batch = 0, cols = 0, numBlocks = 0, blockSize = 0, maxTokens = 0;
};
size_t plan_scratch_ints(int batch);
constexpr int kPlanSlots = 1024; // per workgroup
void launch_plan_blocks(const PlanArgs& a, hipStream_t stream);

struct AddArgs {
    CacheView cache;
    const void* key = nullptr;
    const void* value = nullptr;
    int64_t keyTokenStride = 0, keyHeadStride = 0, valueTokenStride = 0, valueHeadStride = 0; // in elements
    const int* slots = nullptr;
    int* workspace = nullptr; // 3 * numBlocks + 1, where tokens > kAddScan
    int tokens = 0, type = DT_BF16;
};
// more tokens in one call: their blocks are listed (1024 tokens, blocks of 64: 13 us and 39 us without; 256: 11 us either way and
// two launches more)
constexpr int kAddScan = 512;
void launch_cache_add(const AddArgs& a, hipStream_t stream);

struct ReconstructArgs {
    CacheView cache;
    const int* blocks = nullptr;
    void* key = nullptr;   // [n][numHeads][blockSize][headDim]
    void* value = nullptr; // same
    int n = 0, type = DT_F32;
};
void launch_cache_reconstruct(const ReconstructArgs& a, hipStream_t stream);

struct AttendArgs {
    CacheView cache;
    const void* q = nullptr;
    void* out = nullptr;
    float* lse = nullptr; // nullable, [tokens][heads]
    int64_t qTokenStride = 0, qHeadStride = 0, outTokenStride = 0, outHeadStride = 0; // in elements
    const int* table = nullptr;
    int64_t tableStride = 0;
    const int* lengths = nullptr;
    const int* queryOffsets = nullptr; // nullable: one query per request
    int batch = 0, tokens = 0, heads = 0, cols = 0, maxQueries = 0, type = DT_BF16, causal = 1;
    float scale = 1.f;
    void* workspace = nullptr;
    size_t workspaceBytes = 0;
};
size_t cache_attend_workspace(const AttendArgs& a, int num_cus);
int64_t cache_attend_threads(const AttendArgs& a); // of the largest launch, on a whole chip
void launch_cache_attend(const AttendArgs& a, int num_cus, hipStream_t stream);

struct BeamArgs {
    const void* logits = nullptr; // [batch][beams][vocab]
    int64_t batchStride = 0, beamStride = 0;
    const float* scores = nullptr;     // [batch][beams]
    const uint8_t* finished = nullptr; // nullable, [batch][beams]
    float* outScores = nullptr;        // [batch][keep]
    int* parents = nullptr;
    int* tokens = nullptr;
    int batch = 0, beams = 0, keep = 0, padToken = 0, type = DT_F32;
    int64_t vocab = 0;
    void* workspace = nullptr;
    size_t workspaceBytes = 0;
};
constexpr int kMaxBeams = 64; // beams and beams kept
constexpr int kBeamJoin = 1024; // threads that join a batch item's rows
size_t beam_select_workspace(const BeamArgs& a, int num_cus);
void launch_beam_select(const BeamArgs& a, int num_cus, hipStream_t stream);

// rows of `rowBytes` bytes: out[b][j] = in[b][parents[b][j]]
struct ReorderState {
    const void* in;
    void* out;
    int64_t inBatchBytes, inBeamBytes, rowBytes;
};
constexpr int kMaxReorderStates = 64; // per launch
void launch_beam_reorder(const ReorderState* states, int n, const int* parents, int batch, int beams, int keep, hipStream_t stream);

struct ForkArgs {
    const int* table = nullptr;
    int64_t tableStride = 0;
    const int* lengths = nullptr;
    const int* spare = nullptr;
    const int* parents = nullptr; // [batch][beams]
    int* tableOut = nullptr;      // [batch * beams][cols]
    int* lengthsOut = nullptr;
    int* spareOut = nullptr;
    int* owned = nullptr; // nullable: plan_blocks' second table, kept in step
    int64_t ownedStride = 0;
    int batch = 0, beams = 0, cols = 0;
};
constexpr int kMaxForkCaches = 32; // per launch
void launch_fork_blocks(const ForkArgs& a, const CacheView* caches, int n, hipStream_t stream);

// ---- the C entry points' checks of arguments, then the launches above (decoding.cpp)
} // namespace faiss_amd

struct FaissAmdPagedCache;
struct FaissAmdPlanBlocksParams;
struct FaissAmdCacheAddParams;
struct FaissAmdAttendParams;
struct FaissAmdBeamSelectParams;
struct FaissAmdBeamState;
struct FaissAmdForkBlocksParams;
namespace faiss_amd {
class GpuResources;
void plan_blocks(const GpuResources* r, const FaissAmdPlanBlocksParams* p, hipStream_t stream);
void cache_add(const GpuResources* r, const FaissAmdPagedCache* c, const FaissAmdCacheAddParams* p, hipStream_t stream);
void cache_reconstruct(const GpuResources* r, const FaissAmdPagedCache* c, int n, const int* blocks, int type, void* keys, void* values, int checked, hipStream_t stream);
// bytes: no launch, the workspace that the call needs instead
void cache_attend(const GpuResources* r, const FaissAmdPagedCache* c, const FaissAmdAttendParams* p, hipStream_t stream, size_t* bytes);
void beam_select(const GpuResources* r, const FaissAmdBeamSelectParams* p, hipStream_t stream, size_t* bytes);
void reorder_beams(const GpuResources* r, int n, const FaissAmdBeamState* states, const int* parents, int batch, int beams, int keep, int checked, hipStream_t stream);
void fork_blocks(const GpuResources* r, int n, const FaissAmdPagedCache* caches, const FaissAmdForkBlocksParams* p, hipStream_t stream);

} // namespace faiss_amd
