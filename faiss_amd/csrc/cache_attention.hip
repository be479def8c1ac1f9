// faiss_amd/csrc/cache_attention.hip -- attention over a paged cache of 8-bit keys and values.
//
//   o[r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[r] . k_j - m),  k_j = code * kscale[block][head], v_j likewise,
// over the tokens j < len - queries + i + 1 of a request's i-th query (causal; all j < len otherwise).
//
// Both products run on v_mfma_f32_16x16x32_f16: every 8-bit code is an fp16 number exactly (e4m3: 4 significant bits, 2^-9 ...
// 448; int8: integers), fp16 queries are taken as they are, and bf16 queries are shifted by a power of two per row so that their
// largest element lies at 2^10 -- fp16 then holds 24 binades below it exactly, what is lost is 2^-35 of the row's largest element.
// Scores, the running maximum and sum and the accumulators are fp32.  Probabilities are rounded to fp16 (2^-12 relative) after a
// bias of 2^14 in the exponent: they keep their full precision down to 2^-28 of the row's largest, and vanish below 2^-38.
//
// Layout: one wavefront computes S^T = K Q^T for 64 tokens and 16 x NT rows, and O^T += V^T P^T.  Tokens are dealt to the rows of
// the four 16 x 16 score tiles such that lane group g (lanes 16 g ... 16 g + 15) receives exactly the scores of the 16 tokens
// 16 g ... 16 g + 15 of the tile, in order: converted to fp16 they ARE the B operand of the second product, whose A operand
// (V^T: dimension x token) is 16 adjacent bytes of the values' layout.  Nothing goes through LDS or across lanes but the row
// maximum; a block of 16 tokens, the smallest, is one lane group, so a scale is one factor per lane.
#include "decoding.h"
#include <algorithm>

namespace faiss_amd {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 64;        // tokens per step of a wavefront
constexpr int kSeg = 64;         // tiles whose blocks and scales are held in LDS
constexpr float kBias = 6.f, kSlack = 8.f; // see above; both in units of log 2
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// what a launch works on, beside AttendArgs
struct Sched {
    int rowLo, rowHi; // serve the requests with rowLo <= queries * group <= rowHi
    int rows;         // rows of a work item
    int minTiles;     // fewest 64-token tiles of a chunk
    int target;       // chunks are as long as needed to have about this many work items
    int wshift;       // work is counted in units of 2^wshift tiles so that its sum fits an int
    int maxSlots;     // partial results that the workspace holds
    int merge;        // 0: no request is split
    int mergeRows;    // workgroups that join a row tile's rows
    float* partO;     // [maxSlots][rows][dim]
    float2* partML;   // [maxSlots][rows]
};

struct Item {
    int b, h, rt, c, n; // request, head, row tile, chunk, chunks of the request
    int tiles;          // tiles per chunk
    int slot;           // of chunk 0, -1: not split
    int len, q0, nq;    // tokens, first query row and number of queries of the request
};

template <int CODE>
__device__ __forceinline__ half8_t widen(u32x2 w) {
    half2_t r[4];
    if constexpr (CODE == CACHE_E4M3) {
        r[0] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[0], 1.0f, false));
        r[1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[0], 1.0f, true));
        r[2] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[1], 1.0f, false));
        r[3] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[1], 1.0f, true));
    } else {
        // 0x6400 | u is the fp16 number 1024 + u; u = code + 128
        const half2_t off = {(_Float16)1152.f, (_Float16)1152.f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned u = w[i] ^ 0x80808080u;
            r[2 * i] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
            r[2 * i + 1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
        }
    }
    return half8_t{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

// maximum over the four lane groups (lanes with the same lane % 16)
__device__ __forceinline__ float groups_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    x = fmaxf(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)b[0]), __builtin_bit_cast(float, (unsigned)b[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    x = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (unsigned)b[0]) + __builtin_bit_cast(float, (unsigned)b[1]);
}

// the request's queries and tokens, clamped to what the arrays hold whatever the device arrays say
__device__ __forceinline__ void request(const AttendArgs& a, int b, int& len, int& q0, int& nq) {
    const long long cap = (long long)a.cols * a.cache.blockSize;
    len = a.lengths[b];
    len = len < 0 ? 0 : len;
    // tokens behind the table's last column count as bad blocks: one of them is enough to make a row NaN
    len = len > cap ? (int)cap + 1 : len;
    if (a.queryOffsets) {
        q0 = min(max(a.queryOffsets[b], 0), a.tokens);
        nq = min(max(a.queryOffsets[b + 1], q0), a.tokens) - q0;
    } else {
        q0 = b;
        nq = 1;
    }
}

// Deals the work out: chunks of the same number of tiles for every request, so that long and short contexts of a ragged batch
// cost a workgroup the same.  Every wavefront recomputes this from the lengths (a prefix sum over the batch, one step per 64
// requests); a table made by a launch of its own would cost more than it saves.  id: work item (MERGE: row group) number.
template <bool MERGE>
__device__ __forceinline__ bool find_item(const AttendArgs& a, const Sched& s, int id, int xcd_blocks, Item& it) {
    const int lane = threadIdx.x & 63;
    const int G = a.heads / a.cache.numHeads;
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int w = 0;
        if (b < a.batch) {
            int len, q0, nq;
            request(a, b, len, q0, nq);
            const long long rows = (long long)nq * G;
            if (rows >= s.rowLo && rows <= s.rowHi) {
                const long long work = ((rows + s.rows - 1) / s.rows) * (((long long)len + kTile - 1) / kTile);
                w = (int)((work + (1ll << s.wshift) - 1) >> s.wshift);
            }
        }
        sum += __builtin_amdgcn_readlane((int)wave_incl_scan((unsigned)w), 63);
    }
    const long long total = (((long long)sum * a.cache.numHeads) << s.wshift);
    int tiles = (int)min((long long)(1 << 28), (total + s.target - 1) / s.target);
    tiles = max(tiles, s.minTiles);
    // neighbouring items (the row tiles and chunks of one request and head) on one XCD: it.c / it.rt fastest, items dealt in
    // eight contiguous ranges because consecutive workgroups go to the eight XCDs in turn
    int items = 0;
    if (!MERGE && xcd_blocks) {
        for (int b0 = 0; b0 < a.batch; b0 += 64) {
            const int b = b0 + lane;
            int w = 0;
            if (b < a.batch) {
                int len, q0, nq;
                request(a, b, len, q0, nq);
                const long long rows = (long long)nq * G;
                if (rows >= s.rowLo && rows <= s.rowHi) {
                    const int lt = (int)(((long long)len + kTile - 1) / kTile);
                    w = (int)((rows + s.rows - 1) / s.rows) * max(1, (lt + tiles - 1) / tiles) * a.cache.numHeads;
                }
            }
            items += __builtin_amdgcn_readlane((int)wave_incl_scan((unsigned)w), 63);
        }
        const int per = (items + 7) >> 3;
        if ((id >> 3) >= per) return false;
        id = (id & 7) * per + (id >> 3);
        if (id >= items) return false;
    }
    int base = 0, sbase = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int w = 0, sl = 0, len = 0, q0 = 0, nq = 0, n = 1, rts = 0;
        if (b < a.batch) {
            request(a, b, len, q0, nq);
            const long long rows = (long long)nq * G;
            if (rows >= s.rowLo && rows <= s.rowHi) {
                rts = (int)((rows + s.rows - 1) / s.rows);
                const int lt = (int)(((long long)len + kTile - 1) / kTile);
                n = max(1, (lt + tiles - 1) / tiles);
                w = rts * n * a.cache.numHeads;
                sl = n > 1 ? w : 0;
                if (MERGE) w = n > 1 ? rts * a.cache.numHeads : 0;
            }
        }
        const int incl = base + (int)wave_incl_scan((unsigned)w), sincl = sbase + (int)wave_incl_scan((unsigned)sl);
        const unsigned long long hit = __ballot(id < incl);
        if (hit) {
            const int src = __ffsll((long long)hit) - 1;
            const int k = id - __builtin_amdgcn_readlane(incl - w, src);
            it.b = b0 + src;
            it.n = __builtin_amdgcn_readlane(n, src);
            it.len = __builtin_amdgcn_readlane(len, src);
            it.q0 = __builtin_amdgcn_readlane(q0, src);
            it.nq = __builtin_amdgcn_readlane(nq, src);
            rts = __builtin_amdgcn_readlane(rts, src);
            const int s0 = __builtin_amdgcn_readlane(sincl - sl, src);
            it.tiles = tiles;
            if (MERGE) {
                it.c = 0;
                it.rt = k % rts;
                it.h = k / rts;
                it.slot = s0 + k * it.n;
            } else {
                it.c = k % it.n;
                it.rt = (k / it.n) % rts;
                it.h = k / (it.n * rts);
                it.slot = it.n > 1 ? s0 + (k / it.n) * it.n : -1;
            }
            if (it.slot >= 0 && it.slot + it.n > s.maxSlots) return false; // offsets that overlap: nothing to work in
            return true;
        }
        base = __builtin_amdgcn_readlane(incl, 63);
        sbase = __builtin_amdgcn_readlane(sincl, 63);
    }
    return false;
}

// four adjacent elements of a result (any alignment)
__device__ __forceinline__ void store4(unsigned short* p, f32x4 x, float f, int type) {
    unsigned short r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        r[e] = type == DT_F16 ? __builtin_bit_cast(unsigned short, (_Float16)(x[e] * f)) : __builtin_bit_cast(unsigned short, (__bf16)(x[e] * f));
    __builtin_memcpy(p, r, 8);
}

// One work item.  SPLIT: the four wavefronts share the rows and take every fourth tile of the chunk, their results are joined in
// LDS.  Otherwise each has 16 x NT rows of its own and all read the same tiles (through the CU's L1).
template <int D, int CODE, int NT, bool SPLIT>
__global__ __launch_bounds__(256) void cache_attend_kernel(AttendArgs a, Sched s) {
    constexpr int KS = D / 32, MD = D / 16; // steps of the first product, row tiles of the second
    constexpr int NL = D / 64;              // 16-byte pieces of a key per lane (and one of 8 bytes if D % 64)
    constexpr int ROWS = SPLIT ? 16 * NT : 16 * NT * kWaves;
    Item it;
    if (!find_item<false>(a, s, blockIdx.x, 1, it)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n16 = lane & 15, grp = lane >> 4;
    const int H = a.cache.numHeads, G = a.heads / H, bs = a.cache.blockSize;
    const int bsShift = 31 - __builtin_clz(bs);
    const int rowsAll = it.nq * G;
    const int row0 = it.rt * ROWS + (SPLIT ? 0 : wave * 16 * NT);

    // ---- the tiles of this wavefront
    const int lastRow = min(rowsAll, row0 + 16 * NT) - 1;
    int vis = 0, visMin = 0; // tokens that the last / the first row sees
    if (lastRow >= row0) {
        vis = a.causal ? max(0, it.len - it.nq + lastRow / G + 1) : it.len;
        visMin = a.causal ? max(0, it.len - it.nq + row0 / G + 1) : it.len;
    }
    const int step = SPLIT ? kWaves : 1;
    const int tile0 = it.c * it.tiles;
    int tile = tile0 + (SPLIT ? wave : 0);
    const int end = min(tile0 + it.tiles, (vis + kTile - 1) / kTile);
    // what the workgroup's last row sees
    const int lastAll = min(rowsAll, it.rt * ROWS + ROWS) - 1;
    const int visAll = a.causal ? max(0, it.len - it.nq + lastAll / G + 1) : it.len;
    const int endAll = min(tile0 + it.tiles, (visAll + kTile - 1) / kTile);
    // blocks and scales of a stretch of the context, looked up once: a wait for a block's number in the loop would be a wait for
    // all loads issued before it
    __shared__ int pageL[4 * kSeg];
    __shared__ float scaleL[2][4 * kSeg];
    const int* tb = a.table + (int64_t)it.b * a.tableStride;

    // block of the 16 tokens 16 u ...: -1 where there is none, -2 where there should be one
    auto block_of = [&](int u) -> int {
        if (u >= (it.len + 15) >> 4) return -1;
        const int col = (u << 4) >> bsShift;
        if (col >= a.cols) return -2;
        const int p = tb[col];
        return (unsigned)p < (unsigned)a.cache.numBlocks ? p : -2;
    };
    auto look_up = [&](int seg0) {
        for (int i = threadIdx.x; i < 4 * min(kSeg, endAll - seg0); i += 256) {
            const int p = block_of(4 * seg0 + i);
            float ks = p == -2 ? __builtin_nanf("") : 0.f, vs = ks;
            if (p >= 0) {
                ks = a.cache.ks[(int64_t)p * H + it.h];
                vs = a.cache.vs[(int64_t)p * H + it.h];
            }
            pageL[i] = max(p, 0);
            scaleL[0][i] = ks;
            scaleL[1][i] = vs;
        }
    };
    // the codes of a tile, on their way or there
    u32x4 kr[4][NL ? NL : 1];
    u32x2 kx[4];
    u32x4 vr[MD];
    auto fetch_k = [&](int t, int page) {
        const int off = ((t * kTile + 16 * (n16 >> 2)) & (bs - 1)) + (n16 & 3);
        const uint8_t* p = a.cache.k + ((int64_t)page * H + it.h) * (int64_t)(bs * D) + (int64_t)off * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < NL; ++j) kr[i][j] = *(const u32x4*)(p + i * 4 * D + 64 * j + 16 * grp);
            if constexpr (D % 64) kx[i] = *(const u32x2*)(p + i * 4 * D + 64 * NL + 8 * grp);
        }
    };
    auto fetch_v = [&](int t, int page) { // 16 tokens of a dimension per lane
        const uint8_t* p = a.cache.v + ((int64_t)page * H + it.h) * (int64_t)(bs * D) + (int64_t)n16 * bs + ((t * kTile + 16 * grp) & (bs - 1));
#pragma unroll
        for (int i = 0; i < MD; ++i) vr[i] = *(const u32x4*)(p + (int64_t)i * 16 * bs);
    };
    // the first keys are on their way before the queries are looked at
    look_up(tile0);
    __syncthreads();
    if (tile < min(tile0 + kSeg, end)) fetch_k(tile, pageL[(tile - tile0) * 4 + (n16 >> 2)]);

    // ---- queries: lane (n16, grp) holds of row n16 the dimensions 64 j + 16 grp + 8 p ... + 7 for step 2 j + p, the bytes that
    // its lane loads of a key.  qs: what a score is multiplied by beside the block's scale, in units of log 2
    half8_t q[NT][KS];
    float qs[NT];
    int limit[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + n16;
        const bool in = r < rowsAll;
        const int qi = in ? r / G : 0, g = in ? r - qi * G : 0;
        limit[t] = !in ? 0 : a.causal ? max(0, it.len - it.nq + qi + 1) : it.len;
        const int64_t at = (int64_t)(it.q0 + qi) * a.qTokenStride + (int64_t)(it.h * G + g) * a.qHeadStride;
        float x[KS][8];
        float big = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d = (D % 64 && k == KS - 1) ? 64 * NL + 8 * grp : 64 * (k >> 1) + 16 * grp + 8 * (k & 1);
            u32x4 raw; // (any alignment)
            __builtin_memcpy(&raw, (const unsigned short*)a.q + at + d, 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned u = e & 1 ? raw[e >> 1] >> 16 : raw[e >> 1] & 0xffffu;
                float v = a.type == DT_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)u) : __builtin_bit_cast(float, u << 16);
                v = in ? v : 0.f;
                x[k][e] = v;
                const float m = fabsf(v);
                big = (m > big && m < INFINITY) ? m : big;
            }
        }
        float up = 1.f;
        qs[t] = a.scale * kLog2e;
        if (a.type == DT_BF16) {
            big = groups_max(big);
            // largest element to [2^10, 2^11); both factors stay finite: the exponent of a bf16 number is -133 ... 127
            const int e = big > 0.f ? min(max(10 - (int)__builtin_amdgcn_frexp_expf(big), -120), 120) : 0;
            up = __builtin_ldexpf(1.f, e);
            qs[t] *= __builtin_ldexpf(1.f, -e);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[t][k][e] = (_Float16)(x[k][e] * up);
    }

    f32x4 o[NT][MD];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int i = 0; i < MD; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float vref = 0.f, vinv = 0.f; // values are accumulated in units of vref, the largest scale met so far

    auto work = [&](int seg0, int segEnd) {
            const int t0 = tile * kTile;
            const int next = tile + step;
            fetch_v(tile, pageL[(tile - seg0) * 4 + grp]);
            const float ks = scaleL[0][(tile - seg0) * 4 + grp], vs = scaleL[1][(tile - seg0) * 4 + grp];
            // scores
            f32x4 sc4[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int t = 0; t < NT; ++t) sc4[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    u32x2 w;
                    if ((D % 64) && k == KS - 1)
                        w = kx[i];
                    else
                        w = (k & 1) ? u32x2{kr[i][k >> 1][2], kr[i][k >> 1][3]} : u32x2{kr[i][k >> 1][0], kr[i][k >> 1][1]};
                    const half8_t ka = widen<CODE>(w);
#pragma unroll
                    for (int t = 0; t < NT; ++t) sc4[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[t][k], sc4[t][i], 0, 0, 0);
                }
            }
            if (next < segEnd) fetch_k(next, pageL[(next - seg0) * 4 + (n16 >> 2)]);

            // the values' unit
            // (a scale that is no number or has no normal inverse does not become the unit: it must not touch rows that mask it)
            const float va = fabsf(vs);
            const float vmax = groups_max(va >= FLT_MIN && va <= FLT_MAX ? va : 0.f);
            float vdown = 1.f;
            if (vmax > vref) {
                vdown = vref / vmax;
                vref = vmax;
                vinv = 1.f / vmax;
            }
            const float vunit = vs * vinv;
            const bool edge = t0 + kTile > visMin;
            half8_t pr[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float f = ks * qs[t];
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = sc4[t][i][e] * f;
                        if (edge) x = (t0 + 16 * grp + 4 * i + e) < limit[t] ? x : -INFINITY;
                        sc4[t][i][e] = x;
                        mx = fmaxf(mx, x);
                    }
                mx = groups_max(mx);
                // the reference of the exponentials follows the maximum only when that has grown by more than 2^8
                const float mn = mx > m[t] + kSlack ? mx : m[t];
                const float top = mn == -INFINITY ? 0.f : mn;
                const float sub = top - kBias;
                const float down = __builtin_amdgcn_exp2f(m[t] - top);
                m[t] = mn;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float p = __builtin_amdgcn_exp2f(sc4[t][i][e] - sub);
                        sum += p;
                        float pv1 = p * vunit;
                        if (edge) pv1 = p == 0.f ? 0.f : pv1;
                        pr[t][i >> 1][4 * (i & 1) + e] = (_Float16)pv1;
                    }
                l[t] = l[t] * down + sum;
                const float od = down * vdown;
                if (__ballot(od != 1.f)) {
#pragma unroll
                    for (int i = 0; i < MD; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[t][i][e] *= od;
                }
            }
            if (t0 + kTile > it.len) { // what lies behind the last token may be anything, NaN codes too
                const int valid = min(max(it.len - (t0 + 16 * grp), 0), 16);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int nb = min(max(valid - 4 * w, 0), 4);
                    const unsigned mask = nb == 4 ? ~0u : (1u << (8 * nb)) - 1u;
#pragma unroll
                    for (int i = 0; i < MD; ++i) vr[i][w] &= mask;
                }
            }
#pragma unroll
            for (int i = 0; i < MD; ++i) {
                const half8_t a0 = widen<CODE>(u32x2{vr[i][0], vr[i][1]}), a1 = widen<CODE>(u32x2{vr[i][2], vr[i][3]});
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pr[t][0], o[t][i], 0, 0, 0);
                    o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pr[t][1], o[t][i], 0, 0, 0);
                }
            }
            tile = next;
    };
    for (int seg0 = tile0; seg0 < endAll; seg0 += kSeg) {
        const int segEnd = min(seg0 + kSeg, end);
        if (seg0 != tile0) {
            __syncthreads(); // (the segment before has been read)
            look_up(seg0);
            __syncthreads();
            if (tile < segEnd) fetch_k(tile, pageL[(tile - seg0) * 4 + (n16 >> 2)]);
        }
        while (tile < segEnd) work(seg0, segEnd);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) l[t] = groups_sum(l[t]);

    if constexpr (SPLIT) {
        constexpr int PITCH = D + 4;
        __shared__ __align__(16) float sm[kWaves][16 * NT][PITCH];
        __shared__ float sml[kWaves][16 * NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (grp == 0) {
                sml[wave][16 * t + n16][0] = m[t];
                sml[wave][16 * t + n16][1] = l[t];
            }
#pragma unroll
            for (int i = 0; i < MD; ++i) {
                f32x4 x = o[t][i];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] *= vref;
                *(f32x4*)&sm[wave][16 * t + n16][16 * i + 4 * grp] = x;
            }
        }
        __syncthreads();
        // a thread joins 4 dimensions of a row
        for (int x = threadIdx.x; x < 16 * NT * (D / 4); x += 256) {
            const int r = x / (D / 4), d = 4 * (x - r * (D / 4));
            if (row0 + r >= rowsAll) break;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sml[w][r][0]);
            float L = 0.f;
            f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float mw = sml[w][r][0];
                const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
                L += f * sml[w][r][1];
                const f32x4 ow = *(const f32x4*)&sm[w][r][d];
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = __builtin_fmaf(f, ow[e], O[e]);
            }
            if (it.slot >= 0) {
                const int64_t pr = (int64_t)(it.slot + it.c) * ROWS + r;
                *(f32x4*)(s.partO + pr * D + d) = O;
                if (d == 0) s.partML[pr] = make_float2(M, L);
            } else {
                const int qi = (row0 + r) / G, g = (row0 + r) - qi * G;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + d;
                store4(op, O, inv, a.type);
                if (d == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = L == 0.f ? -INFINITY : (M - kBias + __builtin_amdgcn_logf(L)) * kLn2;
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = row0 + 16 * t + n16;
            if (r >= rowsAll) continue;
            if (it.slot >= 0) {
                const int64_t pr = (int64_t)(it.slot + it.c) * ROWS + (r - it.rt * ROWS);
#pragma unroll
                for (int i = 0; i < MD; ++i) {
                    f32x4 x = o[t][i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] *= vref;
                    *(f32x4*)(s.partO + pr * D + 16 * i + 4 * grp) = x;
                }
                if (grp == 0) s.partML[pr] = make_float2(m[t], l[t]);
            } else {
                const int qi = r / G, g = r - qi * G;
                const float inv = l[t] == 0.f ? 0.f : vref / l[t];
                unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + 4 * grp;
#pragma unroll
                for (int i = 0; i < MD; ++i) store4(op + 16 * i, o[t][i], inv, a.type);
                if (grp == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = l[t] == 0.f ? -INFINITY : (m[t] - kBias + __builtin_amdgcn_logf(l[t])) * kLn2;
            }
        }
    }
}

// Joins the chunks of a split request: a workgroup takes every mergeRows-th row.  The chunks' weights come first (all loads in flight together), then
// every group of dim / 4 threads adds up its share of the chunks, eight loads at a time.
constexpr int kMergeChunks = 1024; // weights held at once
__global__ __launch_bounds__(256) void cache_attend_merge_kernel(AttendArgs a, Sched s) {
    Item it;
    if (!find_item<true>(a, s, blockIdx.x / s.mergeRows, 0, it)) return;
    const int D = a.cache.headDim, G = a.heads / a.cache.numHeads;
    for (int r = blockIdx.x % s.mergeRows; r < s.rows; r += s.mergeRows) {
    const int row = it.rt * s.rows + r;
    if (row >= it.nq * G) return;
    __syncthreads();
    const float2* ml = s.partML + (int64_t)it.slot * s.rows + r;
    const float* po = s.partO + ((int64_t)it.slot * s.rows + r) * D;
    const int quads = D / 4, parts = 256 / quads;
    const int part = threadIdx.x / quads, d = 4 * (threadIdx.x - part * quads);
    __shared__ __align__(16) float so[256 * 4];
    __shared__ float wt[kMergeChunks];
    __shared__ float red[2][4];
    float M = -INFINITY;
    for (int c = threadIdx.x; c < it.n; c += 256) M = fmaxf(M, ml[(int64_t)c * s.rows].x);
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < it.n; c0 += kMergeChunks) {
        const int n = min(it.n - c0, kMergeChunks);
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += 256) {
            const float2 x = ml[(int64_t)(c0 + c) * s.rows];
            // a chunk that saw nothing has weight zero and no sums; one of which every score was NaN has a NaN sum
            const float f = x.x == -INFINITY ? (x.y == x.y ? 0.f : x.y) : __builtin_amdgcn_exp2f(x.x - M);
            wt[c] = f;
            L += f == 0.f ? 0.f : f * x.y;
        }
        __syncthreads();
        if (part < parts) {
            const float* p = po + (int64_t)c0 * s.rows * D + d;
            int c = part;
            for (; c + 7 * parts < n; c += 8 * parts) {
                f32x4 v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = *(const f32x4*)(p + (int64_t)(c + e * parts) * s.rows * D);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = wt[c + e * parts];
#pragma unroll
                    for (int j = 0; j < 4; ++j) O[j] = f == 0.f ? O[j] : __builtin_fmaf(f, v[e][j], O[j]);
                }
            }
            for (; c < n; c += parts) {
                const f32x4 v = *(const f32x4*)(p + (int64_t)c * s.rows * D);
                const float f = wt[c];
#pragma unroll
                for (int j = 0; j < 4; ++j) O[j] = f == 0.f ? O[j] : __builtin_fmaf(f, v[j], O[j]);
            }
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o, 64);
    if ((threadIdx.x & 63) == 0) red[1][threadIdx.x >> 6] = L;
    *(f32x4*)&so[4 * threadIdx.x] = O;
    __syncthreads();
    if (threadIdx.x >= quads) continue;
    L = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    for (int p = 1; p < parts; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[e] += so[4 * (p * quads + threadIdx.x) + e];
    const int qi = row / G, g = row - qi * G;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + d;
    store4(op, O, inv, a.type);
    if (d == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = L == 0.f ? -INFINITY : (M - kBias + __builtin_amdgcn_logf(L)) * kLn2;
    }
}

// ------------------------------------------------------------------------------------------------ host side
// rows of a work item and the requests it serves
struct Launch {
    Sched s;
    int nt;
    bool split;
    int64_t grid, mergeGrid;
    size_t bytes;
};

int plan_launches(const AttendArgs& a, int num_cus, Launch out[2]) {
    const int G = a.heads / a.cache.numHeads;
    const int64_t most = (int64_t)a.maxQueries * G;
    int n = 0;
    auto add = [&](int nt, bool split, int lo, int64_t hi) {
        Launch& L = out[n++];
        L.nt = nt;
        L.split = split;
        Sched& s = L.s;
        s.rows = 16 * nt * (split ? 1 : kWaves);
        s.rowLo = lo;
        s.rowHi = (int)std::min<int64_t>(hi, INT32_MAX);
        s.minTiles = split ? 4 : 8;
        s.target = num_cus * (split ? (a.cache.headDim <= 64 ? 6 : a.cache.headDim <= 128 ? 4 : 2) : 2);
        const int64_t rowTiles = ((int64_t)a.tokens * G + s.rows - 1) / s.rows + a.batch;
        const int64_t tiles = ((int64_t)a.cols * a.cache.blockSize + kTile) / kTile;
        s.wshift = 0;
        while (((rowTiles * tiles) >> s.wshift) + a.batch > (int64_t)1 << 30) ++s.wshift;
        s.merge = tiles > s.minTiles;
        // a request with n > 1 chunks has at most twice its share of the total in them
        const int64_t items = s.merge ? 2 * (int64_t)s.target + 2 * (int64_t)a.cache.numHeads : 0;
        s.maxSlots = (int)std::min<int64_t>(items, INT32_MAX);
        L.grid = rowTiles * a.cache.numHeads + items + 8; // (items are dealt to the XCDs in eight ranges of the same length)
        const int64_t groups = std::min<int64_t>(rowTiles * a.cache.numHeads, s.maxSlots / 2);
        s.mergeRows = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(s.rows, most), 8192 / std::max<int64_t>(groups, 1)));
        L.mergeGrid = s.merge ? groups * s.mergeRows : 0;
        L.bytes = s.merge ? round_up((size_t)s.maxSlots * s.rows * a.cache.headDim * 4, 256) + round_up((size_t)s.maxSlots * s.rows * 8, 256) : 0;
        s.partO = nullptr;
        s.partML = nullptr;
    };
    // 256 dimensions and 32 rows do not fit the registers of a wavefront
    const int wide = a.cache.headDim > 192 ? 1 : 2;
    // few rows (single tokens, drafts): the wavefronts of a workgroup split the tokens; many rows: they split the rows
    if (most <= 16) {
        add(1, true, 1, INT64_MAX);
    } else if (most <= 32) {
        add(wide, true, 1, INT64_MAX);
    } else {
        if (a.queryOffsets && G <= 32) add(G <= 16 ? 1 : wide, true, 1, G <= 16 ? 16 : 32);
        add(wide, false, n ? out[0].s.rowHi + 1 : 1, INT64_MAX);
    }
    return n;
}

template <int D, int CODE>
void launch_one(const AttendArgs& a, const Launch& L, hipStream_t stream) {
    const dim3 grid((unsigned)L.grid), block(256);
    // (one row tile without a split of the tokens: only where two do not fit)
    if (L.split && L.nt == 1)
        cache_attend_kernel<D, CODE, 1, true><<<grid, block, 0, stream>>>(a, L.s);
    else if constexpr (D > 192)
        cache_attend_kernel<D, CODE, 1, false><<<grid, block, 0, stream>>>(a, L.s);
    else {
        if (L.split)
            cache_attend_kernel<D, CODE, 2, true><<<grid, block, 0, stream>>>(a, L.s);
        else
            cache_attend_kernel<D, CODE, 2, false><<<grid, block, 0, stream>>>(a, L.s);
    }
    HIP_CHECK(hipGetLastError());
}
template <int D>
void launch_code(const AttendArgs& a, const Launch& L, hipStream_t stream) {
    if (a.cache.code == CACHE_E4M3)
        launch_one<D, CACHE_E4M3>(a, L, stream);
    else
        launch_one<D, CACHE_INT8>(a, L, stream);
}

} // namespace

size_t cache_attend_workspace(const AttendArgs& a, int num_cus) {
    Launch L[2];
    const int n = plan_launches(a, num_cus, L);
    size_t bytes = 0;
    for (int i = 0; i < n; ++i) bytes += L[i].bytes;
    return bytes;
}

void launch_cache_attend(const AttendArgs& a, int num_cus, hipStream_t stream) {
    Launch L[2];
    const int n = plan_launches(a, num_cus, L);
    char* ws = (char*)a.workspace;
    for (int i = 0; i < n; ++i) {
        Sched& s = L[i].s;
        if (s.merge) {
            s.partO = (float*)ws;
            s.partML = (float2*)(ws + round_up((size_t)s.maxSlots * s.rows * a.cache.headDim * 4, 256));
            ws += L[i].bytes;
        }
        FA_THROW_IF_NOT_MSG(L[i].grid < ((int64_t)1 << 31) && L[i].mergeGrid < ((int64_t)1 << 31), "attend: too many rows for one call");
        switch (a.cache.headDim) {
            case 64: launch_code<64>(a, L[i], stream); break;
            case 96: launch_code<96>(a, L[i], stream); break;
            case 128: launch_code<128>(a, L[i], stream); break;
            case 192: launch_code<192>(a, L[i], stream); break;
            case 256: launch_code<256>(a, L[i], stream); break;
            default: FA_THROW_MSG("attend: head dimension not supported");
        }
        if (L[i].mergeGrid > 0) {
            cache_attend_merge_kernel<<<dim3((unsigned)L[i].mergeGrid), dim3(256), 0, stream>>>(a, s);
            HIP_CHECK(hipGetLastError());
        }
    }
}

} // namespace faiss_amd
