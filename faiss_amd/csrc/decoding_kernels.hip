// faiss_amd/csrc/decoding_kernels.hip -- the operators around the attention over a paged cache (decoding.h): block tables and slot
// maps, adding and reading back tokens, beam selection, reordering by parent.
#include "decoding.h"
#include <algorithm>

namespace faiss_amd {
namespace {

typedef unsigned long long u64;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int lane64() {
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
}

// how many bits of the mask stand before this lane's
__device__ __forceinline__ int lanes_before(unsigned long long mask) {
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}

// ================================================================================================ block tables and slot maps
// Requests are served in order.  Request b needs take_b = blocks(new) - blocks(old) more blocks (or returns that many); it is
// granted if the blocks and the slots that the requests up to b ask for together are there.  Both sums only grow with b, so
// the granted requests that add tokens are a prefix of those that ask, and where a request's blocks and slots begin is an
// exclusive prefix sum: one pass.  Free blocks wait in a ring: taken from its front, returned behind its end -- the two ranges
// cannot meet (all blocks together fit the ring), so nothing has to be ordered between requests.  256 requests, a token each: 8 us
// in one workgroup, a chain of dependent loads, 1000 in 11.5; 64 prompts over 384003 slots: 6 + 7 us.  Through the general kernels
// 1025 requests take 32 us, 1500 36, 8000 124: a workgroup goes through them 1024 at a time.
constexpr int kPlanThreads = 1024;

struct PlanScratch { // per request
    int *oldLen, *newLen, *takeStart, *giveStart, *head; // head: {front, count}
};
__host__ __device__ inline PlanScratch plan_scratch(int* p, int batch) {
    return {p, p + batch, p + 2 * batch, p + 3 * batch, p + 4 * batch};
}

// inclusive sums over the workgroup of two non-negative 64-bit values; every thread calls it
__device__ __forceinline__ void wg_scan2(u64& x, u64& y, u64 (*part)[2]) {
    const int lane = lane64(), wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 a = __shfl_up(x, o, 64), b = __shfl_up(y, o, 64);
        if (lane >= o) {
            x += a;
            y += b;
        }
    }
    __syncthreads();
    if (lane == 63) {
        part[wave][0] = x;
        part[wave][1] = y;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        x += part[w][0];
        y += part[w][1];
    }
}

__device__ __forceinline__ int ring_at(int head, u64 i, int n) { // (head + i) mod n, head < n
    u64 p = (u64)head + i;
    if (p >= (u64)n) {
        p -= n;
        if (p >= (u64)n) p %= (u64)n; // (i >= n only where lengths claim more blocks than there are)
    }
    return (int)p;
}

// table entries that request b gains and ring entries that it returns; thread `tid` of `nt`
__device__ __forceinline__ void plan_fill_blocks(const PlanArgs& a, const PlanScratch& s, int b, int tid, int nt) {
    if (!a.granted[b]) return;
    const int bs = a.blockSize;
    const int have = (s.oldLen[b] + bs - 1) / bs, want = (s.newLen[b] + bs - 1) / bs;
    const int head = s.head[0], count = s.head[1];
    int* row = a.table + (int64_t)b * a.tableStride;
    int* own = a.owned ? a.owned + (int64_t)b * a.ownedStride : nullptr;
    for (int i = have + tid; i < want; i += nt) {
        const int p = a.ring[ring_at(head, (u64)s.takeStart[b] + (i - have), a.numBlocks)];
        row[i] = p;
        if (own) own[i] = p;
    }
    for (int i = want + tid; i < have; i += nt)
        a.ring[ring_at(head, (u64)count + s.giveStart[b] + (i - want), a.numBlocks)] = own ? own[i] : row[i];
}

// slot of the t-th new token of the call
__device__ __forceinline__ int plan_slot(const PlanArgs& a, const PlanScratch& s, int t) {
    if (t >= a.queryOffsets[a.batch]) return -1;
    int lo = 0, hi = a.batch; // last request that starts at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.queryOffsets[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    const int bs = a.blockSize;
    const int pos = s.oldLen[lo] + (t - a.queryOffsets[lo]), col = pos / bs, have = (s.oldLen[lo] + bs - 1) / bs;
    const int p = col >= have ? a.ring[ring_at(s.head[0], (u64)s.takeStart[lo] + (col - have), a.numBlocks)]
                              : a.table[(int64_t)lo * a.tableStride + col];
    return (unsigned)p < (unsigned)a.numBlocks ? p * bs + (pos - col * bs) : -1;
}

// All of it in one workgroup, for batches of up to a thread per request: sums of 32 bits (a request asks for no more than one block
// or slot beyond what there is -- it is refused then either way), what the requests hold is kept in LDS, and the blocks and slots
// of the call are dealt to the threads one by one.
constexpr int kPlanSmallTokens = 1 << 20; // (1024 requests of them fit 32 bits)
struct PlanLds {
    int oldLen[kPlanThreads], newLen[kPlanThreads];
    int take[kPlanThreads + 1], give[kPlanThreads + 1], off[kPlanThreads + 1]; // where a request's blocks and slots begin
};
// last request that begins at or before t
__device__ __forceinline__ int plan_owner(const int* start, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}
__device__ __forceinline__ int wg_scan(int x, int* part) { // inclusive, every thread calls it
    const int lane = lane64(), wave = threadIdx.x >> 6;
    x = (int)wave_incl_scan((unsigned)x);
    __syncthreads();
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = lane < wave ? part[lane] : 0; // (at most 16 wavefronts)
    before = __builtin_amdgcn_readlane((int)wave_incl_scan((unsigned)before), 63);
    return x + before;
}

// FILL: the table and the slots too (few tokens); else what plan_fill_kernel goes by
template <bool FILL>
__global__ __launch_bounds__(kPlanThreads) void plan_small_kernel(PlanArgs a) {
    __shared__ PlanLds z;
    __shared__ int part[kPlanThreads / 64], top[2];
    const int b = threadIdx.x, bs = a.blockSize, N = a.numBlocks;
    const unsigned cap = (unsigned)a.cols * (unsigned)bs;
    int oldLen = 0, newLen = 0;
    if (b < a.batch) {
        oldLen = a.lengths[b];
        newLen = a.newLengths[b];
    }
    long long h0 = a.state[0];
    const long long count = min(max((long long)a.state[1], 0ll), (long long)N);
    if (h0 < 0 || h0 >= N) h0 = ((h0 % N) + N) % N;
    const int head = (int)h0;
    if (b < 2) top[b] = 0;
    const bool ok = b < a.batch && (unsigned)oldLen <= cap && (unsigned)newLen <= cap;
    const int have = ok ? (int)(((unsigned)oldLen + bs - 1) / bs) : 0, want = ok ? (int)(((unsigned)newLen + bs - 1) / bs) : 0;
    const int tok = ok ? min(max(newLen - oldLen, 0), a.maxTokens + 1) : 0, need = min(max(want - have, 0), a.maxTokens + 1);
    const int ct = wg_scan(need, part), cn = wg_scan(tok, part);
    const bool granted = ok && (tok == 0 || (ct <= count && cn <= a.maxTokens));
    if (granted && tok > 0) {
        atomicMax(&top[0], ct);
        atomicMax(&top[1], cn);
    }
    const int mine = granted ? max(have - want, 0) : 0;
    const int give = wg_scan(mine, part); // (its barriers order the maxima)
    const int taken = top[0], placed = top[1];
    if (b < a.batch) {
        z.oldLen[b] = oldLen;
        z.newLen[b] = newLen;
        // (a refused request begins where the granted ones end: nothing is its own)
        z.take[b] = min(ct - need, taken);
        z.off[b] = min(cn - tok, placed);
        z.give[b] = give - mine;
        a.granted[b] = granted;
        a.lengthsOut[b] = granted ? newLen : oldLen;
        a.queryOffsets[b] = z.off[b];
        if (b == a.batch - 1) {
            z.give[a.batch] = give;
            z.take[a.batch] = taken;
            z.off[a.batch] = placed;
        }
    }
    if (a.batch == 0 && b == 0) z.give[0] = z.take[0] = z.off[0] = 0;
    __syncthreads();
    const int given = z.give[a.batch];
    if (b == 0) {
        a.queryOffsets[a.batch] = placed;
        a.stateOut[0] = ring_at(head, taken, N);
        a.stateOut[1] = min(count - taken + given, (long long)N);
    }
    if (!FILL) {
        const PlanScratch s = plan_scratch(a.scratch, a.batch);
        if (b < a.batch) {
            s.oldLen[b] = oldLen;
            s.newLen[b] = newLen;
            s.takeStart[b] = z.take[b];
            s.giveStart[b] = z.give[b];
        }
        if (b == 0) {
            s.head[0] = head;
            s.head[1] = (int)count;
        }
        return;
    }
    for (int t = threadIdx.x; t < taken; t += kPlanThreads) {
        const int r = plan_owner(z.take, a.batch, t), col = (z.oldLen[r] + bs - 1) / bs + (t - z.take[r]);
        const int p = a.ring[ring_at(head, t, N)];
        a.table[(int64_t)r * a.tableStride + col] = p;
        if (a.owned) a.owned[(int64_t)r * a.ownedStride + col] = p;
    }
    for (int t = threadIdx.x; t < given; t += kPlanThreads) {
        const int r = plan_owner(z.give, a.batch, t), col = (z.newLen[r] + bs - 1) / bs + (t - z.give[r]);
        a.ring[ring_at(head, (u64)count + t, N)] = a.owned ? a.owned[(int64_t)r * a.ownedStride + col] : a.table[(int64_t)r * a.tableStride + col];
    }
    for (int t = threadIdx.x; t < a.maxTokens; t += kPlanThreads) {
        int slot = -1;
        if (t < placed) {
            const int r = plan_owner(z.off, a.batch, t), pos = z.oldLen[r] + (t - z.off[r]), col = pos / bs, first = (z.oldLen[r] + bs - 1) / bs;
            const int p = col >= first ? a.ring[ring_at(head, z.take[r] + (col - first), N)] : a.table[(int64_t)r * a.tableStride + col];
            if ((unsigned)p < (unsigned)N) slot = p * bs + (pos - col * bs);
        }
        a.slots[t] = slot;
    }
}

// batches of any size
__global__ __launch_bounds__(kPlanThreads) void plan_scan_kernel(PlanArgs a) {
    __shared__ u64 part[kPlanThreads / 64][2];
    __shared__ u64 tot[2];
    const PlanScratch s = plan_scratch(a.scratch, a.batch);
    const int bs = a.blockSize;
    const long long cap = (long long)a.cols * bs;
    long long h0 = a.state[0] % a.numBlocks;
    if (h0 < 0) h0 += a.numBlocks;
    const long long count = min(max((long long)a.state[1], 0ll), (long long)a.numBlocks);
    u64 takeBase = 0, tokBase = 0, giveBase = 0, taken = 0, placed = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
        const int b = b0 + threadIdx.x;
        int oldLen = 0, newLen = 0, need = 0, tok = 0;
        bool ok = false;
        if (b < a.batch) {
            oldLen = a.lengths[b];
            newLen = a.newLengths[b];
            ok = oldLen >= 0 && newLen >= 0 && oldLen <= cap && newLen <= cap;
            if (ok) {
                need = (int)(((long long)newLen + bs - 1) / bs) - (int)(((long long)oldLen + bs - 1) / bs);
                tok = max(newLen - oldLen, 0);
            }
        }
        u64 ct = need > 0 ? need : 0, cn = tok;
        wg_scan2(ct, cn, part);
        ct += takeBase;
        cn += tokBase;
        const bool granted = ok && (tok == 0 || (ct <= (u64)count && cn <= (u64)a.maxTokens));
        // totals of the granted requests: sums up to the last one that adds
        u64 give = granted && need < 0 ? -need : 0, dummy = 0;
        const u64 ownGive = give;
        __syncthreads();
        if (threadIdx.x == 0) tot[0] = tot[1] = 0;
        wg_scan2(give, dummy, part); // (its barriers order the reset)
        if (granted && tok > 0) {
            atomicMax(&tot[0], ct);
            atomicMax(&tot[1], cn);
        }
        __syncthreads();
        taken = max(taken, tot[0]);
        placed = max(placed, tot[1]);
        if (b < a.batch) {
            s.oldLen[b] = oldLen;
            s.newLen[b] = newLen;
            s.takeStart[b] = (int)min(ct - (need > 0 ? need : 0), (u64)INT32_MAX);
            s.giveStart[b] = (int)min(giveBase + give - ownGive, (u64)INT32_MAX);
            a.granted[b] = granted;
            a.lengthsOut[b] = granted ? newLen : oldLen;
            // (a refused request starts where the granted ones end: it has no tokens)
            a.queryOffsets[b] = (int)min(cn - tok, placed);
        }
        // running totals: the last thread's sums
        __syncthreads();
        if (threadIdx.x == kPlanThreads - 1) {
            part[0][0] = ct;
            part[0][1] = cn;
            part[1][0] = giveBase + give;
        }
        __syncthreads();
        takeBase = part[0][0];
        tokBase = part[0][1];
        giveBase = part[1][0];
    }
    if (threadIdx.x == 0) {
        s.head[0] = (int)h0;
        s.head[1] = (int)count;
        a.queryOffsets[a.batch] = (int)placed;
        a.stateOut[0] = ring_at((int)h0, taken, a.numBlocks);
        a.stateOut[1] = min(count - (long long)taken + (long long)giveBase, (long long)a.numBlocks);
    }
}

__global__ __launch_bounds__(256) void plan_fill_kernel(PlanArgs a) {
    const PlanScratch s = plan_scratch(a.scratch, a.batch);
    if ((int)blockIdx.x < a.batch) {
        plan_fill_blocks(a, s, blockIdx.x, threadIdx.x, 256);
        return;
    }
    const int64_t t0 = (int64_t)(blockIdx.x - a.batch) * kPlanSlots;
    for (int64_t t = t0 + threadIdx.x; t < min(t0 + kPlanSlots, (int64_t)a.maxTokens); t += 256) a.slots[t] = plan_slot(a, s, (int)t);
}

// ================================================================================================ adding and reading tokens
// scale of a (block, head) = the smallest power of two with which its largest element stays in the codes' range.  Powers of two:
// a block whose scale has to grow is re-expressed without a division, exactly in e4m3 (but for the last codes above zero), and an
// element is rounded once when it is added -- with scales of amax / range every growth would round all older codes anew.  The
// price is in int8, half a bit of the step on average (at most one); e4m3 has the same relative step at every scale.
constexpr int kMaxBlockSize = 256;

template <int CODE>
__device__ __forceinline__ float pow2_scale(unsigned amax_bits) { // bits of a finite |x|
    if (amax_bits == 0) return 0.f;
    const int top = CODE == CACHE_E4M3 ? 8 : 6;                                // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
    const unsigned frac = CODE == CACHE_E4M3 ? 0x600000u : 0x7e0000u;
    int e = (int)(amax_bits >> 23) - 127 - top + ((amax_bits & 0x7fffffu) > frac ? 1 : 0);
    e = max(e, -126);
    return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}
template <int CODE>
__device__ __forceinline__ unsigned encode4(float x0, float x1, float x2, float x3) {
    if constexpr (CODE == CACHE_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    } else {
        // x + 1.5 * 2^23 is rounded to an integer (half to even) that stands in the low bits, in two's complement
        const float r = 12582912.f;
        const unsigned a = __builtin_bit_cast(unsigned, x0 + r), b = __builtin_bit_cast(unsigned, x1 + r);
        const unsigned c = __builtin_bit_cast(unsigned, x2 + r), d = __builtin_bit_cast(unsigned, x3 + r);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
    }
}
template <int CODE>
__device__ __forceinline__ void decode4(unsigned w, float x[4]) {
    if constexpr (CODE == CACHE_E4M3) {
        x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int)(signed char)(w >> (8 * i));
    }
}
// the four codes of a word multiplied by ratio < 1 and rounded
template <int CODE>
__device__ __forceinline__ unsigned rescale4(unsigned w, float ratio) {
    float x[4];
    decode4<CODE>(w, x);
    return encode4<CODE>(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
}
// four words of four bytes, transposed: byte j of word i becomes byte i of word j
__device__ __forceinline__ void transpose4(unsigned w[4]) {
    const unsigned a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const unsigned c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}
// eight adjacent elements of 16 bits; VEC: they are 16-byte aligned
template <bool VEC>
__device__ __forceinline__ u32x4 elems8(const void* p, int64_t at) {
    if (VEC) return *(const u32x4*)((const unsigned short*)p + at);
    unsigned short u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = ((const unsigned short*)p)[at + i];
    u32x4 r;
    __builtin_memcpy(&r, u, 16);
    return r;
}
template <int CODE>
__device__ __forceinline__ u32x2 encode8(u32x4 raw, int type, float inv) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned lo = raw[i] & 0xffffu, hi = raw[i] >> 16;
        x[2 * i] = (type == DT_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)lo) : __builtin_bit_cast(float, lo << 16)) * inv;
        x[2 * i + 1] = (type == DT_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)hi) : __builtin_bit_cast(float, hi << 16)) * inv;
    }
    return u32x2{encode4<CODE>(x[0], x[1], x[2], x[3]), encode4<CODE>(x[4], x[5], x[6], x[7])};
}

// The blocks of a call: found[0] of them, found[1 + i] (in no particular order: they are independent), and where the tokens of block
// b begin and end, spans[2 * b] and spans[2 * b + 1].  Two launches, since the entries of the call's blocks, and only those, are set
// (FIRST) before the tokens meet in them.
template <bool FIRST>
__global__ __launch_bounds__(256) void add_blocks_kernel(AddArgs a) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    int* spans = a.workspace;
    int* found = a.workspace + 2 * (int64_t)a.cache.numBlocks;
    if (FIRST && j == 0) found[0] = 0;
    if (j >= a.tokens) return;
    const int shift = 31 - __builtin_clz(a.cache.blockSize);
    const int mine = a.slots[j], block = mine >> shift;
    if (mine < 0 || block >= a.cache.numBlocks) return;
    const bool begins = j == 0 || a.slots[j - 1] >> shift != block, ends = j == a.tokens - 1 || a.slots[j + 1] >> shift != block;
    if (FIRST) {
        if (begins) spans[2 * block] = 0x7fffffff, spans[2 * block + 1] = -1;
    } else {
        if (begins && atomicMin(&spans[2 * block], j) == 0x7fffffff) found[1 + atomicAdd(found, 1)] = block;
        if (ends) atomicMax(&spans[2 * block + 1], j);
    }
}

// blockIdx.y: the keys or the values of a head.  A workgroup of few tokens (LISTED false) looks at token blockIdx.x: where its block
// differs from its predecessor's it scans the call's slots for all tokens of that block: if none comes earlier it serves them (a
// block's tokens may stand anywhere in the call; of several tokens for one slot the last wins), else another workgroup does.  Many
// tokens would be scanned too often (65536 tokens in blocks of 64: 8.6 ms): for them the blocks are listed first, and a
// workgroup takes every gridDim.x-th, and scans from its first token to its last.
// Keys are written as 8 dimensions of a token, values as 4 tokens of 8 dimensions: 4 x 4 bytes are transposed in registers, so
// that both layouts get words.  16384 tokens of 8 x 128, int8, blocks of 64: 33 us with the list (100 MB, 20 us at the rate of a
// copy), 65536: 109 us; 256 tokens of as many blocks of 16: 8.5 us in a graph (9.7 under a tracer), of 64 18, of 128 26, 4096 tokens of
// as many blocks of 64 240: a value's code is a byte in a line of its own.
template <int CODE, bool VEC, int NT, bool LISTED>
__global__ __launch_bounds__(NT) void cache_add_kernel(AddArgs a) {
    const CacheView& c = a.cache;
    const int bs = c.blockSize, D = c.headDim, H = c.numHeads, oct = D / 8;
    const int64_t nslots = (int64_t)c.numBlocks * bs;
    const int lane = threadIdx.x & 63, tid = threadIdx.x;
    __shared__ __align__(16) int token[kMaxBlockSize];
    __shared__ int earlier;
    __shared__ unsigned part[NT / 64];
    const int shift = 31 - __builtin_clz(bs);
    const int* found = a.workspace + 2 * (int64_t)c.numBlocks;
    const int count = LISTED ? found[0] : a.tokens;
    for (int n = blockIdx.x; n < count; n += gridDim.x) {
        int block, me = n, to = a.tokens;
        if constexpr (LISTED) {
            block = found[1 + n];
            me = a.workspace[2 * block];
            to = a.workspace[2 * block + 1] + 1;
        } else {
            const int mine = a.slots[n];
            block = mine >> shift;
            if (mine < 0 || mine >= nslots || (n > 0 && a.slots[n - 1] >> shift == block)) continue;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < bs; i += NT) token[i] = -1;
        if (threadIdx.x == 0) earlier = 0;
        __syncthreads();
        const int first = block * bs;
        for (int j0 = (LISTED ? me : 0) + threadIdx.x; j0 < to; j0 += 8 * NT) { // eight loads in flight: the scan is latency, not bytes
            int s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = j0 + NT * e < to ? a.slots[j0 + NT * e] : -1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = j0 + NT * e;
                const unsigned o = (unsigned)(s[e] - first); // (-1 - first >= bs as an unsigned number)
                if (o < (unsigned)bs) {
                    atomicMax(&token[o], j);
                    if (j < me) earlier = 1;
                }
            }
        }
        __syncthreads();
        if (earlier) continue;
        const bool fresh = token[0] >= 0;
        const int unit = blockIdx.y;
        const bool isV = unit >= H;
        const int h = isV ? unit - H : unit;
        const void* x = isV ? a.value : a.key;
        const int64_t ts = isV ? a.valueTokenStride : a.keyTokenStride, base = (int64_t)h * (isV ? a.valueHeadStride : a.keyHeadStride);
        // a thread's piece: 4 tokens x 8 dimensions; neighbours hold the next dimensions (keys), the next tokens (values)
        const int quads = bs / 4, pieces = quads * oct; // (pieces <= 2048: i / oct by a reciprocal is exact)
        const unsigned recip = 65536 / oct + 1;
        auto piece = [&](int i, int& q, int& o) {
            q = isV ? i & (quads - 1) : (int)((i * recip) >> 16);
            o = isV ? i >> (shift - 2) : i - q * oct;
        };
        auto load = [&](int q, int o, u32x4 (&raw)[4]) { // (false: none of the four is in the call)
            const int4 t = *(const int4*)&token[4 * q];
            const int tt[4] = {t.x, t.y, t.z, t.w};
            if (max(max(tt[0], tt[1]), max(tt[2], tt[3])) < 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[e] = u32x4{0u, 0u, 0u, 0u};
                return false;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = elems8<VEC>(x, base + max(tt[e], me) * ts + 8 * o);
            if (min(min(tt[0], tt[1]), min(tt[2], tt[3])) < 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[e] = tt[e] >= 0 ? raw[e] : u32x4{0u, 0u, 0u, 0u};
            }
            return true;
        };
        // largest element: sixteen bits without the sign order like the numbers
        u32x4 raw[4];
        u16x2 most = {0, 0};
        for (int i = tid; i < pieces; i += NT) {
            int q, o;
            piece(i, q, o);
            if (!load(q, o, raw)) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, raw[e][w] & 0x7fff7fffu));
        }
        unsigned big = max(most[0], most[1]);
#pragma unroll
        for (int o = 32; o; o >>= 1) big = max(big, (unsigned)__shfl_xor((int)big, o, 64));
        if (lane == 0) part[tid >> 6] = big;
        float* sp = (isV ? c.vs : c.ks) + (int64_t)block * H + h;
        const float old = *sp;
        __syncthreads(); // (and every thread has read the old scale)
        for (int w = 0; w < NT / 64; ++w) big = max(big, part[w]);
        const float amax = a.type == DT_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)big) : __builtin_bit_cast(float, big << 16);
        const float before = fresh ? 0.f : old;
        float after = __builtin_nanf("");
        // anything that is no number makes the block's scale, and with it all its values, no number until the block is begun anew
        if (amax < INFINITY && before >= 0.f && before < INFINITY) after = fmaxf(before, pow2_scale<CODE>(__builtin_bit_cast(unsigned, amax)));
        const bool number = after == after;
        // (a subnormal scale is one that the caller has brought, and all that is added is zero: its inverse may be infinite)
        const float inv = number && after >= FLT_MIN ? 1.f / after : 0.f;
        const float ratio = after > 0.f ? before / after : 0.f;
        const bool rescale = fresh || (number && ratio != 1.f), clear = rescale && ratio == 0.f;
        uint8_t* codes = (isV ? c.v : c.k) + ((int64_t)block * H + h) * (int64_t)bs * D;
        for (int i = tid; i < pieces; i += NT) {
            int q, o;
            piece(i, q, o);
            const int4 t = *(const int4*)&token[4 * q];
            const int tt[4] = {t.x, t.y, t.z, t.w};
            unsigned mask = 0; // tokens that are written
#pragma unroll
            for (int e = 0; e < 4; ++e) mask |= tt[e] >= 0 ? 0xffu << (8 * e) : 0u;
            if (!mask && !rescale) continue;
            if (pieces > NT) load(q, o, raw); // (else it is still there)
            u32x2 w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = number ? encode8<CODE>(raw[e], a.type, inv) : u32x2{0u, 0u};
            if (!isV) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    u32x2* p = (u32x2*)(codes + (int64_t)(4 * q + e) * D + 8 * o);
                    if (tt[e] < 0) {
                        if (!rescale) continue;
                        if (!clear) {
                            const u32x2 was = *p;
                            w[e] = u32x2{rescale4<CODE>(was[0], ratio), rescale4<CODE>(was[1], ratio)};
                        }
                    }
                    *p = w[e];
                }
            } else {
                unsigned lo[4] = {w[0][0], w[1][0], w[2][0], w[3][0]}, hi[4] = {w[0][1], w[1][1], w[2][1], w[3][1]};
                transpose4(lo);
                transpose4(hi);
                unsigned* p = (unsigned*)(codes + (int64_t)(8 * o) * bs + 4 * q);
                unsigned was[8];
                if (mask != ~0u && !clear) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) was[e] = p[e * (bs / 4)];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    unsigned now = e < 4 ? lo[e & 3] : hi[e & 3];
                    if (mask != ~0u && !clear) now = (now & mask) | ((rescale ? rescale4<CODE>(was[e], ratio) : was[e]) & ~mask);
                    p[e * (bs / 4)] = now;
                }
            }
        }
        if (tid == 0) *sp = after;
    }
}

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ _Float16 narrow<_Float16>(float x) { return (_Float16)x; }
template <>
__device__ __forceinline__ __bf16 narrow<__bf16>(float x) { return (__bf16)x; }

template <int CODE, typename T>
__device__ __forceinline__ void store8(T* p, unsigned lo, unsigned hi, float scale) {
    float x[8];
    decode4<CODE>(lo, x);
    decode4<CODE>(hi, x + 4);
    T r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = narrow<T>(x[e] * scale);
    __builtin_memcpy(__builtin_assume_aligned(p, 16), r, 8 * sizeof(T));
}

// a workgroup per (block, head), the keys or the values of it (blockIdx.y); the values' bytes are transposed as cache_add_kernel does.
// Bound by memory: 262 blocks of 8 x 64 x 128, keys and values, to fp16 in 19 us (103 MB, 5.4 TB/s)
template <int CODE, typename T>
__global__ __launch_bounds__(256) void cache_reconstruct_kernel(ReconstructArgs a) {
    const CacheView& c = a.cache;
    const int bs = c.blockSize, D = c.headDim, H = c.numHeads, oct = D / 8;
    const int i = blockIdx.x / H, h = blockIdx.x - i * H;
    const int block = a.blocks[i];
    const bool isV = blockIdx.y == 1;
    T* out = (T*)(isV ? a.value : a.key) + (int64_t)blockIdx.x * bs * D;
    const bool none = (unsigned)block >= (unsigned)c.numBlocks; // no such block: no such values
    const int64_t at = none ? 0 : (int64_t)block * H + h;
    const float scale = none ? __builtin_nanf("") : isV ? c.vs[at] : c.ks[at];
    const uint8_t* codes = (isV ? c.v : c.k) + at * bs * D;
    if (!isV) {
        for (int x = threadIdx.x; x < bs * oct; x += 256) {
            const u32x2 w = *(const u32x2*)(codes + 8 * x);
            store8<CODE>(out + 8 * x, w[0], w[1], scale);
        }
    } else {
        const int quads = bs / 4;
        for (int x = threadIdx.x; x < quads * oct; x += 256) {
            const int q = x / oct, o = x - q * oct;
            unsigned lo[4], hi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo[e] = *(const unsigned*)(codes + (int64_t)(8 * o + e) * bs + 4 * q);
                hi[e] = *(const unsigned*)(codes + (int64_t)(8 * o + 4 + e) * bs + 4 * q);
            }
            transpose4(lo);
            transpose4(hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) store8<CODE>(out + (int64_t)(4 * q + e) * D + 8 * o, lo[e], hi[e], scale);
        }
    }
}

// ================================================================================================ beam selection
// value(w, v) = score_w + x_wv - log sum_v exp x_wv.  Inside a beam candidates rank as their logits do, so one pass over the logits
// keeps the `keep` best (logit, lowest v) of every piece of a row beside its maximum and sum of exponentials; a second launch
// joins the pieces of a row, then the rows of a batch item.  An exponential is an fp32 one: its argument is off by (2^-23 + 2^-26)
// |x - max|, the instruction by 2^-23; four are added in fp32, everything beyond that in 64 bits, and candidates of different beams are
// compared as 64-bit values.  Measured, a log-sum is off by 1e-8 where logits are spread (128001 of them, 3e-8 at 1000) and by up
// to 8e-8 where one dominates (all sixteen of a lane added in fp32, and lanes joined by fp32 exponentials: 6e-8 and 9e-7, in the
// same time); beams whose values are closer than that may change places.
// 512 rows of 128001 bf16 logits, 16 kept: 44 us (131 MB, 3.0 TB/s) and 9 us for the join; 4 rows of 32000:
// 8 + 5 us.  13.5 vector instructions per logit keep the SIMDs busy for half of the time; neither they nor the memory are full.
constexpr int kBeamVpt = 16;                                   // logits per lane and step
constexpr int kBeamPend = 128;                                 // keys a wavefront collects before it cuts them to `keep`
constexpr int kBeamCap = kBeamPend + 64 * kBeamVpt / 2;        // keys a wavefront may hold at once
constexpr int kBeamKeys = 2048;                                // keys of a row that the second launch joins

struct BeamSched {
    int parts;
    u64* keys;    // [rows][parts][keep]
    double* sums; // [rows][parts]
    float* maxs;  // [rows][parts]
};

// (ordkey, index) of a logit: smaller is better; ~0 for what is no candidate
__device__ __forceinline__ u64 beam_key(float x, unsigned v) {
    return x > -INFINITY ? ((u64)~float_flip(x) << 32) | v : ~0ull;
}
__device__ __forceinline__ float beam_logit(u64 key) { return float_unflip(~(unsigned)(key >> 32)); }

// A bound that exactly `keep` of the n unique keys in LDS do not exceed (n > keep): bits from the top, a ballot per 64 keys and
// bit.  The low half, which only tells equal logits apart, is looked at where they straddle the bound.
template <int R>
__device__ __forceinline__ u64 wave_kth_regs(const u64* list, int n, int keep) {
    const int lane = lane64();
    unsigned hi[R], lo[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const u64 k = 64 * r + lane < n ? list[64 * r + lane] : ~0ull;
        hi[r] = (unsigned)(k >> 32);
        lo[r] = (unsigned)k;
    }
    unsigned t = 0;
    for (int b = 31; b >= 0; --b) {
        const unsigned c = t | ((1u << b) - 1);
        int cnt = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) cnt += __popcll(__ballot(hi[r] <= c));
        if (cnt < keep) t |= 1u << b;
    }
    int below = 0, upto = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        below += __popcll(__ballot(hi[r] < t));
        upto += __popcll(__ballot(hi[r] <= t));
    }
    if (upto == keep) return ((u64)t << 32) | ~0u;
    unsigned u = 0;
    for (int b = 31; b >= 0; --b) {
        const unsigned c = u | ((1u << b) - 1);
        int cnt = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) cnt += __popcll(__ballot(hi[r] == t && lo[r] <= c));
        if (cnt < keep - below) u |= 1u << b;
    }
    return ((u64)t << 32) | u;
}
__device__ __forceinline__ u64 wave_kth(const u64* list, int n, int keep) {
    if (n <= 64) return wave_kth_regs<1>(list, n, keep);
    if (n <= 128) return wave_kth_regs<2>(list, n, keep);
    if (n <= 256) return wave_kth_regs<4>(list, n, keep);
    const int lane = lane64();
    u64 t = 0;
    for (int b = 63; b >= 0; --b) {
        const u64 c = t | ((1ull << b) - 1);
        int cnt = 0;
        for (int i = lane; i < n; i += 64) cnt += list[i] <= c;
        cnt = __builtin_amdgcn_readlane((int)wave_incl_scan((unsigned)cnt), 63);
        if (cnt < keep) t |= 1ull << b;
    }
    return t;
}
// keeps the keys <= kth of the n in LDS, in place
__device__ __forceinline__ int wave_cut(u64* list, int n, u64 kth) {
    const int lane = lane64();
    int out = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const u64 k = i0 + lane < n ? list[i0 + lane] : ~0ull;
        const bool in = i0 + lane < n && k <= kth;
        const u64 m = __ballot(in);
        __builtin_amdgcn_wave_barrier();
        if (in) list[out + __popcll(m & ((1ull << lane) - 1))] = k;
        out += __popcll(m);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    return out;
}

template <typename T, int ROUND>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamArgs a, BeamSched s) {
    constexpr int PER = 16 / sizeof(T); // logits of a 16-byte load
    constexpr int LD = kBeamVpt / PER;
    __shared__ __align__(16) u64 lists[4][kBeamCap];
    __shared__ unsigned short groups[4][64 * ROUND];
    __shared__ double ss[4];
    __shared__ float sm[4];
    __shared__ int sn[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x / s.parts;
    const int part = (int)(blockIdx.x - row * s.parts);
    const int bi = (int)(row / a.beams), w = (int)(row - (int64_t)bi * a.beams);
    const int keep = a.keep;
    u64* out = s.keys + (row * s.parts + part) * keep;
    if (a.finished && a.finished[row]) { // its one candidate is made by the second launch
        if (threadIdx.x < keep) out[threadIdx.x] = ~0ull;
        return;
    }
    const T* x = (const T*)a.logits + (int64_t)bi * a.batchStride + (int64_t)w * a.beamStride;
    // granules of 16 bytes from the row's first logit, shared out to the parts and wavefronts in runs of 64 x LD.  By index and not
    // by address: rows of the same logits then have the same sum to the last bit wherever they lie, and equal beams stay tied
    // (the loads need no alignment)
    const int64_t granules = (a.vocab + PER - 1) / PER;
    const int64_t steps = (granules + 64 * LD - 1) / (64 * LD);
    u64* list = lists[wave];
    int n = 0;
    float thr = -FLT_MAX; // only logits of at least this can be among the best (-inf is no candidate)
    bool full = false;    // the list holds `keep` logits that are no smaller
    float m = -INFINITY;
    double sum = 0.0;
    const int64_t stride = (int64_t)s.parts * 4;
    auto fetch = [&](int64_t st, int l, T (&to)[kBeamVpt]) { // the logits of a lane in a step
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int64_t e0 = ((st * LD + i) * 64 + l) * PER;
            if (e0 + PER <= a.vocab) {
                __builtin_memcpy(to + i * PER, x + e0, 16);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e) to[i * PER + e] = e0 + e < a.vocab ? x[e0 + e] : (T)-INFINITY;
            }
        }
    };
    T next[kBeamVpt];
    int64_t st = (int64_t)part * 4 + wave;
    if (st < steps) fetch(st, lane, next);
    // ROUND steps at a time: their sums and the largest logit of every lane in every step; then, from what is still in the
    // caches, the few lanes' logits again whose largest can be among the best
    for (; st < steps; st += ROUND * stride) {
        float best[ROUND];
#pragma unroll
        for (int j = 0; j < ROUND; ++j) {
            best[j] = -INFINITY;
            if (st + j * stride < steps) {
                float v[kBeamVpt];
#pragma unroll
                for (int i = 0; i < kBeamVpt; ++i) v[i] = (float)next[i];
                if (st + (j + 1) * stride < steps) fetch(st + (j + 1) * stride, lane, next);
                float mx = v[0];
#pragma unroll
                for (int i = 1; i < kBeamVpt; ++i) mx = fmaxf(mx, v[i]);
                best[j] = mx;
                // running maximum and sum of the lane; a NaN or an infinity makes the sum NaN
                const float mn = fmaxf(m, mx);
                double p = 0.0;
#pragma unroll
                for (int i = 0; i < kBeamVpt; i += 4) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) e[j] = __builtin_amdgcn_exp2f((v[i + j] - mn) * 1.4426950408889634f);
                    p += (double)((e[0] + e[1]) + (e[2] + e[3])); // (one that dominates leaves the others 24 bits, not 20)
                }
                if (mn == -INFINITY) { // (nothing but -inf so far, or a NaN among it)
                    float q = 0.f;
#pragma unroll
                    for (int i = 0; i < kBeamVpt; ++i) q = v[i] == v[i] ? q : v[i];
                    sum += (double)q;
                } else {
                    sum = sum * (double)__builtin_amdgcn_exp2f((m - mn) * 1.4426950408889634f) + p;
                }
                m = mn;
            }
        }
        if (!full) {
            // the keep-th best of the lanes' best logits (of their upper 16 bits, rounded down) bounds the keep best
            unsigned k[ROUND], t = 0;
#pragma unroll
            for (int j = 0; j < ROUND; ++j) k[j] = best[j] > -INFINITY ? ~float_flip(best[j]) >> 16 : 0xffffu;
            for (int b = 15; b >= 0; --b) {
                const unsigned c = t | ((1u << b) - 1);
                int cnt = 0;
#pragma unroll
                for (int j = 0; j < ROUND; ++j) cnt += __popcll(__ballot(k[j] <= c));
                if (cnt < keep) t |= 1u << b;
            }
            thr = fmaxf(float_unflip(~((t << 16) | 0xffffu)), -FLT_MAX); // (NaN where there are fewer: -FLT_MAX)
        }
        int ng = 0;
#pragma unroll
        for (int j = 0; j < ROUND; ++j) {
            const u64 mask = __ballot(best[j] >= thr);
            if (best[j] >= thr) groups[wave][ng + lanes_before(mask)] = (unsigned short)(64 * j + lane);
            ng += __popcll(mask);
        }
        if (!ng) continue;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        for (int g0 = 0; g0 < ng; g0 += 64) {
            const bool is = g0 + lane < ng;
            const int g = groups[wave][min(g0 + lane, ng - 1)];
            const int64_t gs = st + (g >> 6) * stride;
            T again[kBeamVpt];
            fetch(gs, g & 63, again);
            const unsigned first = (unsigned)((gs * LD * 64 + (g & 63)) * PER); // index of the first of them
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (n > kBeamPend) n = wave_cut(list, n, wave_kth(list, n, keep));
#pragma unroll
                for (int j = 0; j < kBeamVpt / 2; ++j) {
                    const int i = half * (kBeamVpt / 2) + j;
                    const float v = (float)again[i];
                    const bool in = is && v >= thr;
                    const u64 mask = __ballot(in);
                    if (!mask) continue;
                    if (in) list[n + lanes_before(mask)] = beam_key(v, first + (unsigned)(64 * PER * (i / PER) + i % PER));
                    n += __popcll(mask);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            }
        }
        if (n > keep) {
            const u64 kth = wave_kth(list, n, keep);
            n = wave_cut(list, n, kth);
            thr = beam_logit(kth);
            full = true;
        }
    }
    if (n > keep) n = wave_cut(list, n, wave_kth(list, n, keep));
    // the wavefront's maximum and sum, then the workgroup's
    float M = m;
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    double S = (m == -INFINITY && sum == sum) ? 0.0 : sum * exp((double)m - (double)M);
#pragma unroll
    for (int o = 32; o; o >>= 1) S += __shfl_xor(S, o, 64);
    if (lane == 0) {
        sm[wave] = M;
        ss[wave] = S;
        sn[wave] = n;
    }
    __syncthreads();
    if (wave) return;
    // wavefront 0 appends the others' lists to its own (4 keep <= 256 keys)
    for (int o = 1; o < 4; ++o) {
        const int no = sn[o];
        for (int i = lane; i < no; i += 64) list[n + i] = lists[o][i];
        n += no;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    if (n > keep) n = wave_cut(list, n, wave_kth(list, n, keep));
    for (int i = lane; i < keep; i += 64) out[i] = i < n ? list[i] : ~0ull;
    if (lane == 0) {
        float MM = -INFINITY;
        for (int o = 0; o < 4; ++o) MM = fmaxf(MM, sm[o]);
        double SS = 0.0;
        for (int o = 0; o < 4; ++o)
            if (sm[o] > -INFINITY || ss[o] != ss[o]) SS += ss[o] * exp((double)sm[o] - (double)MM);
        s.maxs[row * s.parts + part] = MM;
        s.sums[row * s.parts + part] = SS;
    }
}

__device__ __forceinline__ u64 double_flip(double x) { // larger is smaller
    const u64 u = __builtin_bit_cast(u64, x == 0.0 ? 0.0 : x);
    return ~((u >> 63) ? ~u : (u | (1ull << 63)));
}

// a workgroup of 16 wavefronts per batch item
__global__ __launch_bounds__(kBeamJoin) void beam_join_kernel(BeamArgs a, BeamSched s) {
    __shared__ u64 val[kMaxBeams * kMaxBeams]; // double_flip of a candidate's value
    __shared__ unsigned tok[kMaxBeams * kMaxBeams];
    __shared__ int ranks[kMaxBeams * kMaxBeams];
    __shared__ int valid;
    __shared__ u64 lists[kBeamJoin / 64][256 + kMaxBeams];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, keep = a.keep, b = blockIdx.x;
    const int total = a.beams * keep;
    for (int i = threadIdx.x; i < total; i += kBeamJoin) ranks[i] = 0;
    if (threadIdx.x == 0) valid = 0;
    for (int w = wave; w < a.beams; w += kBeamJoin / 64) {
        const int64_t row = (int64_t)b * a.beams + w;
        const u64* keys = s.keys + row * s.parts * keep;
        const int count = s.parts * keep;
        // (the loads do not wait for one another: the launch is latency)
        const bool fin = a.finished && a.finished[row];
        const double score = (double)a.scores[row];
        float pm = lane < s.parts ? s.maxs[row * s.parts + lane] : -INFINITY;
        double ps = lane < s.parts ? s.sums[row * s.parts + lane] : 0.0;
        u64 first[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) first[j] = 64 * j + lane < count ? keys[64 * j + lane] : ~0ull;
        u64* vw = val + w * keep;
        unsigned* tw = tok + w * keep;
        if (fin) {
            for (int i = lane; i < keep; i += 64) {
                vw[i] = i == 0 && score > -INFINITY ? double_flip(score) : ~0ull;
                tw[i] = (unsigned)a.padToken;
            }
            continue;
        }
        // log of the sum of the row's exponentials
        float M = pm;
        for (int p = lane + 64; p < s.parts; p += 64) M = fmaxf(M, s.maxs[row * s.parts + p]);
#pragma unroll
        for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        double S = 0.0;
        for (int p = lane; p < s.parts; p += 64) {
            if (p >= 64) {
                pm = s.maxs[row * s.parts + p];
                ps = s.sums[row * s.parts + p];
            }
            if (pm > -INFINITY || ps != ps) S += ps * exp((double)pm - (double)M);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) S += __shfl_xor(S, o, 64);
        const double lse = (double)M + log(S);
        // the row's best, cut in LDS four times 64 keys at a time
        u64* list = lists[wave];
        int n = 0;
        u64 thr = ~0ull;
        for (int i0 = 0; i0 < count; i0 += 256) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + 64 * j + lane;
                const u64 k = i0 == 0 ? first[j] : i < count ? keys[i] : ~0ull;
                const bool in = k < thr;
                const u64 mask = __ballot(in);
                if (in) list[n + __popcll(mask & ((1ull << lane) - 1))] = k;
                n += __popcll(mask);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            if (n > keep) {
                thr = wave_kth(list, n, keep);
                n = wave_cut(list, n, thr);
            }
        }
        for (int i = lane; i < keep; i += 64) {
            u64 v = ~0ull;
            unsigned t = 0;
            if (i < n) {
                const double value = score + ((double)beam_logit(list[i]) - lse);
                if (value > -INFINITY) v = double_flip(value); // (NaN: no candidate)
                t = (unsigned)list[i];
            }
            vw[i] = v;
            tw[i] = t;
        }
    }
    __syncthreads();
    // rank of each candidate among those of the batch item: by value, then beam, then token.  A thread compares one candidate
    // with the candidates of every `share`-th beam
    const int share = max(1, min(kBeamJoin / total, a.beams));
    for (int x = threadIdx.x; x < total * share; x += kBeamJoin) {
        const int i = x / share, g = x - i * share, w = i / keep;
        const u64 v = val[i];
        if (v == ~0ull) continue;
        const unsigned t = tok[i];
        int rank = 0;
        for (int ow = g; ow < a.beams; ow += share)
            for (int j = ow * keep; j < (ow + 1) * keep; ++j) {
                const u64 o = val[j];
                rank += o < v || (o == v && (ow < w || (ow == w && tok[j] < t)));
            }
        if (rank) atomicAdd(&ranks[i], rank);
        if (g == 0) atomicAdd(&valid, 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += kBeamJoin) {
        const u64 v = val[i];
        const int rank = ranks[i];
        if (v == ~0ull || rank >= keep) continue;
        const int64_t at = (int64_t)b * keep + rank;
        const u64 u = ~v;
        a.outScores[at] = (float)__builtin_bit_cast(double, (u >> 63) ? (u & ~(1ull << 63)) : ~u);
        a.parents[at] = i / keep;
        a.tokens[at] = (int)tok[i];
    }
    for (int i = valid + threadIdx.x; i < keep; i += kBeamJoin) { // fewer candidates than asked for
        const int64_t at = (int64_t)b * keep + i;
        a.outScores[at] = -INFINITY;
        a.parents[at] = -1;
        a.tokens[at] = -1;
    }
}

// ================================================================================================ reordering by parent
struct ReorderPiece { // `bytes` of a state's rows, from in and out on
    const uint8_t* in;
    uint8_t* out;
    int64_t inBatchBytes, inBeamBytes, rowBytes, bytes;
};
template <int CAP>
struct ReorderTable { // (a kernel's argument: a launch of few states carries few)
    ReorderPiece st[CAP];
    int first[CAP + 1]; // workgroups of a row before piece i
};
constexpr int kReorderBytes = 16384; // of a row per workgroup

// 80 rows of 147 KB in six states of odd lengths: 6.2 us (24 MB; byte by byte 17.7 us)
template <int CAP>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderTable<CAP> tab, int n, const int* parents, int beams, int keep) {
    const int chunk = blockIdx.y;
    int lo = 0;
    while (lo + 1 < n && tab.first[lo + 1] <= chunk) ++lo;
    const ReorderPiece& s = tab.st[lo];
    const int64_t row = blockIdx.x;
    const int b = (int)(row / keep);
    const int parent = parents[row];
    const int64_t at = (int64_t)(chunk - tab.first[lo]) * kReorderBytes, len = min((int64_t)kReorderBytes, s.bytes - at);
    uint8_t* out = s.out + row * s.rowBytes + at;
    const bool none = parent < 0 || parent >= beams; // such a row becomes zero
    const uint8_t* in = s.in + (int64_t)b * s.inBatchBytes + (int64_t)(none ? 0 : parent) * s.inBeamBytes + at;
    // rows of any length lie anywhere: 16 bytes at a time where the output is aligned (the loads need not be), single ones around
    const int head = (int)min(len, (int64_t)((16 - ((uintptr_t)out & 15)) & 15)), mid = (int)(len - head) / 16, done = head + 16 * mid;
    u32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = threadIdx.x + 256 * j;
        v[j] = u32x4{0u, 0u, 0u, 0u};
        if (i < mid && !none) __builtin_memcpy(&v[j], in + head + 16 * i, 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = threadIdx.x + 256 * j;
        if (i < mid) *(u32x4*)(out + head + 16 * i) = v[j];
    }
    const int edge = threadIdx.x < 16 ? threadIdx.x : done + threadIdx.x - 16;
    if (threadIdx.x < 16 ? edge < head : edge < len) out[edge] = none ? 0 : in[edge];
}

struct ForkTable {
    CacheView c[kMaxForkCaches];
};
// blockIdx.x: row; blockIdx.y: 0 the table, 1 + i cache i.  A copy: 256 rows x 8 caches x 131 KB in 105 us (5.1 TB/s)
__global__ __launch_bounds__(256) void fork_blocks_kernel(ForkArgs a, ForkTable tab, int blockSize, int numBlocks, int withTable) {
    const int row = blockIdx.x, b = row / a.beams;
    int parent = a.parents[row];
    parent = parent < 0 || parent >= a.beams ? row : b * a.beams + parent;
    const int cap = a.cols * blockSize;
    const int len = min(max(a.lengths[parent], 0), cap), mine = min(max(a.lengths[row], 0), cap);
    const int tail = len % blockSize ? len / blockSize : -1; // column of the parent's partly filled block
    const int src = tail >= 0 ? a.table[(int64_t)parent * a.tableStride + tail] : -1;
    const int dst = a.spare[row];
    const bool ok = tail >= 0 && (unsigned)src < (unsigned)numBlocks && (unsigned)dst < (unsigned)numBlocks;
    if (withTable && blockIdx.y == 0) {
        for (int j = threadIdx.x; j < a.cols; j += 256)
            a.tableOut[(int64_t)row * a.cols + j] = j == tail ? (ok ? dst : -1) : a.table[(int64_t)parent * a.tableStride + j];
        if (threadIdx.x == 0) {
            a.lengthsOut[row] = a.lengths[parent];
            int spare = tail < 0 ? dst : mine % blockSize ? a.table[(int64_t)row * a.tableStride + mine / blockSize] : -1;
            if (a.owned) { // the row's blocks and its spare one change places: each block stays in one of the two
                spare = dst;
                if (ok) {
                    int* own = a.owned + (int64_t)row * a.ownedStride + tail;
                    spare = *own;
                    *own = dst;
                }
            }
            a.spareOut[row] = spare;
        }
        return;
    }
    if (!ok) return;
    const CacheView& c = tab.c[blockIdx.y - withTable];
    const int64_t bytes = (int64_t)c.numHeads * blockSize * c.headDim;
    const u32x4 *k = (const u32x4*)(c.k + src * bytes), *v = (const u32x4*)(c.v + src * bytes);
    u32x4 *ko = (u32x4*)(c.k + dst * bytes), *vo = (u32x4*)(c.v + dst * bytes);
    for (int64_t i = threadIdx.x; i < bytes / 16; i += 256) {
        ko[i] = k[i];
        vo[i] = v[i];
    }
    for (int h = threadIdx.x; h < c.numHeads; h += 256) {
        c.ks[(int64_t)dst * c.numHeads + h] = c.ks[(int64_t)src * c.numHeads + h];
        c.vs[(int64_t)dst * c.numHeads + h] = c.vs[(int64_t)src * c.numHeads + h];
    }
}

void beam_sched(const BeamArgs& a, int num_cus, BeamSched& s, size_t& bytes) {
    const int64_t rows = (int64_t)a.batch * a.beams;
    // about eight workgroups per CU, each wavefront a step of its own, and no more keys of a row than its join takes at once
    int64_t parts = (8 * (int64_t)num_cus + rows - 1) / std::max<int64_t>(rows, 1);
    parts = std::min<int64_t>(parts, (a.vocab + 4 * 64 * kBeamVpt - 1) / (4 * 64 * kBeamVpt));
    parts = std::min<int64_t>(parts, kBeamKeys / a.keep);
    s.parts = (int)std::max<int64_t>(parts, 1);
    const size_t kb = round_up((size_t)rows * s.parts * a.keep * 8, 256), sb = round_up((size_t)rows * s.parts * 8, 256);
    char* p = (char*)a.workspace;
    s.keys = (u64*)p;
    s.sums = (double*)(p + kb);
    s.maxs = (float*)(p + kb + sb);
    bytes = kb + sb + round_up((size_t)rows * s.parts * 4, 256);
}

} // namespace

size_t plan_scratch_ints(int batch) { return (size_t)batch * 4 + 2; }

void launch_plan_blocks(const PlanArgs& a, hipStream_t stream) {
    // (cols: what a request returns is summed in 32 bits too)
    const bool small = a.batch <= kPlanThreads && a.maxTokens <= kPlanSmallTokens && a.cols <= 1 << 20;
    const bool fill = small && a.maxTokens <= 4 * kPlanThreads;
    if (fill)
        plan_small_kernel<true><<<1, kPlanThreads, 0, stream>>>(a);
    else if (small)
        plan_small_kernel<false><<<1, kPlanThreads, 0, stream>>>(a);
    else
        plan_scan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
    HIP_CHECK(hipGetLastError());
    if (fill) return;
    plan_fill_kernel<<<(unsigned)(a.batch + div_up(a.maxTokens, kPlanSlots)), 256, 0, stream>>>(a);
    HIP_CHECK(hipGetLastError());
}

template <int CODE>
static void launch_add(const AddArgs& a, bool vec, hipStream_t stream) {
    const bool listed = a.tokens > kAddScan;
    const int units = 2 * a.cache.numHeads;
    // a workgroup per token of few (with four tokens each, 512 in a row in blocks of 64 take 13 us instead of 21 and 300 7 instead of
    // 10, but a decoding step of as many 37 instead of 32 and 25 instead of 21, and those come more often); of many, four times as many workgroups of 256 threads as the chip holds, so that blocks even out
    const dim3 grid((unsigned)(listed ? std::min(a.tokens, std::max(8192 / units, 1)) : a.tokens), units);
    if (listed) {
        const unsigned n = (unsigned)div_up(a.tokens, 256);
        add_blocks_kernel<true><<<n, 256, 0, stream>>>(a);
        add_blocks_kernel<false><<<n, 256, 0, stream>>>(a);
    }
    // a wavefront per workgroup where a block has a piece for each lane (64 x 128, a token: 6 us with four wavefronts, 11 with one)
    const bool small = a.cache.blockSize * a.cache.headDim / 32 <= 64;
    auto launch = [&](auto kernel, int nt) { kernel<<<grid, nt, 0, stream>>>(a); };
    if (!vec)
        listed ? launch(cache_add_kernel<CODE, false, 256, true>, 256) : launch(cache_add_kernel<CODE, false, 256, false>, 256);
    else if (small)
        listed ? launch(cache_add_kernel<CODE, true, 64, true>, 64) : launch(cache_add_kernel<CODE, true, 64, false>, 64);
    else
        listed ? launch(cache_add_kernel<CODE, true, 256, true>, 256) : launch(cache_add_kernel<CODE, true, 256, false>, 256);
}
void launch_cache_add(const AddArgs& a, hipStream_t stream) {
    if (a.tokens == 0) return;
    const bool vec = ((uintptr_t)a.key | (uintptr_t)a.value) % 16 == 0 &&
            (a.keyTokenStride | a.keyHeadStride | a.valueTokenStride | a.valueHeadStride) % 8 == 0;
    if (a.cache.code == CACHE_E4M3)
        launch_add<CACHE_E4M3>(a, vec, stream);
    else
        launch_add<CACHE_INT8>(a, vec, stream);
    HIP_CHECK(hipGetLastError());
}

template <int CODE>
static void launch_reconstruct(const ReconstructArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((int64_t)a.n * a.cache.numHeads), 2);
    if (a.type == DT_F32)
        cache_reconstruct_kernel<CODE, float><<<grid, 256, 0, stream>>>(a);
    else if (a.type == DT_F16)
        cache_reconstruct_kernel<CODE, _Float16><<<grid, 256, 0, stream>>>(a);
    else
        cache_reconstruct_kernel<CODE, __bf16><<<grid, 256, 0, stream>>>(a);
}
void launch_cache_reconstruct(const ReconstructArgs& a, hipStream_t stream) {
    if (a.n == 0) return;
    if (a.cache.code == CACHE_E4M3)
        launch_reconstruct<CACHE_E4M3>(a, stream);
    else
        launch_reconstruct<CACHE_INT8>(a, stream);
    HIP_CHECK(hipGetLastError());
}

size_t beam_select_workspace(const BeamArgs& a, int num_cus) {
    BeamSched s;
    size_t bytes;
    beam_sched(a, num_cus, s, bytes);
    return bytes;
}
template <typename T>
static void launch_beam_scan(const BeamArgs& a, const BeamSched& s, unsigned grid, hipStream_t stream) {
    // eight steps between two selections, one where a wavefront has no more than two (4 x 32000 logits: 7.9 us against 10.5;
    // 512 x 128001: 54 us with one, 43 with eight)
    const int64_t step = 64 * kBeamVpt, per = 4 * (int64_t)s.parts * step;
    if (a.vocab <= 2 * per)
        beam_scan_kernel<T, 1><<<grid, 256, 0, stream>>>(a, s);
    else
        beam_scan_kernel<T, 8><<<grid, 256, 0, stream>>>(a, s);
}
void launch_beam_select(const BeamArgs& a, int num_cus, hipStream_t stream) {
    if (a.batch == 0) return;
    BeamSched s;
    size_t bytes;
    beam_sched(a, num_cus, s, bytes);
    const int64_t grid = (int64_t)a.batch * a.beams * s.parts;
    if (a.type == DT_F32)
        launch_beam_scan<float>(a, s, (unsigned)grid, stream);
    else if (a.type == DT_F16)
        launch_beam_scan<_Float16>(a, s, (unsigned)grid, stream);
    else
        launch_beam_scan<__bf16>(a, s, (unsigned)grid, stream);
    HIP_CHECK(hipGetLastError());
    beam_join_kernel<<<a.batch, kBeamJoin, 0, stream>>>(a, s);
    HIP_CHECK(hipGetLastError());
}

// Pieces of up to 65535 chunks go into a launch (a grid has no more in y), and long rows into several
void launch_beam_reorder(const ReorderState* states, int n, const int* parents, int batch, int beams, int keep, hipStream_t stream) {
    const int64_t rows = (int64_t)batch * keep;
    if (rows == 0) return;
    constexpr int FEW = 8, ROOM = 65535;
    ReorderTable<kMaxReorderStates> tab;
    int k = 0, chunks = 0;
    auto launch = [&]() {
        if (k == 0) return;
        tab.first[k] = chunks;
        const dim3 grid((unsigned)rows, (unsigned)chunks);
        if (k <= FEW) {
            ReorderTable<FEW> few;
            std::copy(tab.st, tab.st + k, few.st);
            std::copy(tab.first, tab.first + k + 1, few.first);
            beam_reorder_kernel<FEW><<<grid, 256, 0, stream>>>(few, k, parents, beams, keep);
        } else {
            beam_reorder_kernel<kMaxReorderStates><<<grid, 256, 0, stream>>>(tab, k, parents, beams, keep);
        }
        HIP_CHECK(hipGetLastError());
        k = chunks = 0;
    };
    for (int i = 0; i < n; ++i)
        for (int64_t at = 0; at < states[i].rowBytes;) {
            if (k == kMaxReorderStates || chunks == ROOM) launch();
            ReorderPiece& p = tab.st[k];
            p.in = (const uint8_t*)states[i].in + at;
            p.out = (uint8_t*)states[i].out + at;
            p.inBatchBytes = states[i].inBatchBytes;
            p.inBeamBytes = states[i].inBeamBytes;
            p.rowBytes = states[i].rowBytes;
            p.bytes = std::min(states[i].rowBytes - at, (int64_t)(ROOM - chunks) * kReorderBytes);
            tab.first[k++] = chunks;
            chunks += (int)((p.bytes + kReorderBytes - 1) / kReorderBytes);
            at += p.bytes;
        }
    launch();
}

void launch_fork_blocks(const ForkArgs& a, const CacheView* caches, int n, hipStream_t stream) {
    const int rows = a.batch * a.beams;
    if (rows == 0) return;
    const int bs = caches[0].blockSize, nb = caches[0].numBlocks;
    for (int i = 0; i == 0 || i < n; i += kMaxForkCaches) {
        ForkTable tab;
        const int m = std::min(kMaxForkCaches, n - i);
        for (int j = 0; j < m; ++j) tab.c[j] = caches[i + j];
        fork_blocks_kernel<<<dim3((unsigned)rows, (unsigned)(m + (i == 0))), 256, 0, stream>>>(a, tab, bs, nb, i == 0);
        HIP_CHECK(hipGetLastError());
    }
}

} // namespace faiss_amd
