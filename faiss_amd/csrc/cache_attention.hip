// faiss_amd/csrc/cache_attention.hip -- attention over a paged cache of 8-bit keys and values.
//
//   o[r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[r] . k_j - m),  k_j = code * kscale[block][head], v_j likewise,
// over the tokens j < len - queries + i + 1 of a request's i-th query (causal; all j < len otherwise).
//
// Both products run on v_mfma_f32_16x16x32_f16: every 8-bit code is an fp16 number exactly (e4m3: 4 significant bits, 2^-9 ...
// 448; int8: integers), fp16 queries are taken as they are, and bf16 queries are shifted by a power of two per row so that their
// largest element lies in [2^9, 2^10) -- fp16 then holds 23 binades below it exactly, what is lost is 2^-34 of the row's largest
// element.  Scores, the running reference and sum and the accumulators are fp32.  A probability is rounded to fp16 (2^-11 relative)
// together with its value's scale, in units in which the largest such product of the row lies between 2^6 and 2^14: it keeps its
// precision down to 2^-20 of that, and vanishes below 2^-31.
//
// Layout: one wavefront computes S^T = K Q^T for 64 tokens and 16 x NT rows, and O^T += V^T P^T.  Tokens are dealt to the rows of
// the four 16 x 16 score tiles such that lane group g (lanes 16 g ... 16 g + 15) receives exactly the scores of the 16 tokens
// 16 g ... 16 g + 15 of the tile, in order: converted to fp16 they ARE the B operand of the second product, whose A operand
// (V^T: dimension x token) is 16 adjacent bytes of the values' layout.  Nothing goes across lanes but the row maximum; a block of
// 16 tokens, the smallest, is one lane group, so a scale is one factor per lane.
//
// Two kernels feed these products: straight from memory for few rows (bound by the cache's bytes), through LDS for many (bound by
// the arithmetic); a third joins the chunks of split contexts.
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
constexpr float kNoScale = -1000.f;
constexpr float kNothing = -FLT_MAX; // reference of a row that has seen nothing (finite: its differences are no NaN)
constexpr int kSeg = 64;         // tiles whose blocks and scales are held in LDS
constexpr float kBias = 6.f, kSlack = 8.f; // see above; both in units of log 2
constexpr float kRoom = 40.f;    // what the sums of probabilities are kept below their reference, see softmax_step
constexpr float kFar = 4096.f;   // references beyond this are taken from a base of their own, see softmax_step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// what a launch works on, beside AttendArgs
struct Sched {
    int rowLo, rowHi; // serve the requests with rowLo <= queries * group <= rowHi
    int rows, rowShift; // rows of a work item, 2^rowShift
    int minTiles;     // fewest 64-token tiles of a chunk
    int target;       // chunks are as long as needed to have about this many work items
    int slack;        // a request is split only if it is this many times as long as a chunk
    int wshift;       // work is counted in units of 2^wshift tiles so that its sum fits an int
    int maxSlots;     // partial results that the workspace holds
    int merge;        // 0: no request is split
    int sort;         // of 64 requests, the longest first
    int mergeRows;    // workgroups that join a row tile's rows
    float* partO;     // [maxSlots][rows][dim]: results of chunks
    float4* partML;   // [maxSlots][rows]: {base, reference, sum} of their probabilities
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
// the larger, NaN if either is: one instruction, where fmaxf first quiets the operands that come from a matrix instruction (a row of
// which a score is NaN becomes NaN whatever its reference)
__device__ __forceinline__ float highest(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float groups_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    x = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (unsigned)b[0]) + __builtin_bit_cast(float, (unsigned)b[1]);
}

// the request's queries and tokens, clamped to what the arrays hold whatever the device arrays say
__device__ __forceinline__ void request(const AttendArgs& a, int b, int& len, int& q0, int& nq) {
    len = max(a.lengths[b], 0);
    if (a.queryOffsets) {
        q0 = min(max(a.queryOffsets[b], 0), a.tokens);
        nq = min(max(a.queryOffsets[b + 1], q0), a.tokens) - q0;
    } else {
        q0 = b;
        nq = 1;
    }
}

__device__ __forceinline__ int tiles_of(int len) { return (int)(((unsigned)len + kTile - 1) / kTile); }
// tiles that are worked on.  Tokens behind the table's last column count as bad blocks: the first of them makes every row NaN that
// sees any (the rows' limits go by the length as it is)
__device__ __forceinline__ int tiles_within(const AttendArgs& a, int len) { return tiles_of(min(len, a.cols * a.cache.blockSize + 1)); }
__device__ __forceinline__ int chunks(int lt, int tiles, int slack) {
    return (unsigned)lt > (unsigned)tiles * slack ? (lt + tiles - 1) / tiles : 1;
}

// Deals the work out: chunks of the same number of tiles for every request, so that long and short contexts of a ragged batch
// cost a workgroup the same.  Every wavefront recomputes this from the lengths (a prefix sum over the batch, one step per 64
// requests); a table made by a launch of its own would cost more than it saves.  id: work item (MERGE: row group) number.
template <bool MERGE>
__device__ __forceinline__ bool find_item(const AttendArgs& a, const Sched& s, int id, Item& it) {
    const int lane = threadIdx.x & 63;
    const int G = a.heads / a.cache.numHeads;
    // (tokens x heads fits an int, and the host chose wshift for the sums)
    auto row_tiles = [&](int nq) {
        const int rows = nq * G;
        return rows >= s.rowLo && rows <= s.rowHi ? (rows + s.rows - 1) >> s.rowShift : 0;
    };
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int w = 0;
        if (b < a.batch) {
            int len, q0, nq;
            request(a, b, len, q0, nq);
            const long long work = (long long)row_tiles(nq) * tiles_within(a, len);
            w = (int)((work + (1ll << s.wshift) - 1) >> s.wshift);
        }
        sum += __builtin_amdgcn_readlane((int)wave_incl_scan((unsigned)w), 63);
    }
    // (a division of floats: the same in every wavefront, and what it is off by is within the slack of maxSlots)
    const float share = ceilf((float)sum * (float)a.cache.numHeads * __builtin_ldexpf(1.f, s.wshift) / (float)s.target);
    const int tiles = max((int)fminf(share, 0x1p28f), s.minTiles);
    // Consecutive workgroups go to the eight XCDs in turn, so every XCD gets its share of every request; the heads of a row tile
    // follow one another, the row tiles that see most come first, and of 64 requests the longest.
    int base = 0, sbase = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        int b = b0 + lane;
        if (s.sort && b0 + 1 < a.batch) {
            const int key = b < a.batch ? a.lengths[b] : -1; // (any order would do)
            int rank = 0;
            for (int j = 0; j < min(64, a.batch - b0); ++j) {
                const int o = __builtin_amdgcn_readlane(key, j);
                rank += o > key || (o == key && j < lane);
            }
            if (b < a.batch) b = b0 + rank;
            b = __builtin_amdgcn_ds_permute(4 * (b - b0), lane) + b0;
        }
        int w = 0, sl = 0, len = 0, q0 = 0, nq = 0, n = 1, rts = 0;
        if (b < a.batch) {
            request(a, b, len, q0, nq);
            rts = row_tiles(nq);
            n = chunks(tiles_within(a, len), tiles, s.slack);
            w = rts * n * a.cache.numHeads;
            sl = n > 1 ? w : 0;
            if (MERGE) w = n > 1 ? rts * a.cache.numHeads : 0;
        }
        const int incl = base + (int)wave_incl_scan((unsigned)w), sincl = sbase + (int)wave_incl_scan((unsigned)sl);
        const unsigned long long hit = __ballot(id < incl);
        if (hit) {
            const int src = __ffsll((long long)hit) - 1;
            const int k = id - __builtin_amdgcn_readlane(incl - w, src);
            it.b = __builtin_amdgcn_readlane(b, src);
            it.n = __builtin_amdgcn_readlane(n, src);
            it.len = __builtin_amdgcn_readlane(len, src);
            it.q0 = __builtin_amdgcn_readlane(q0, src);
            it.nq = __builtin_amdgcn_readlane(nq, src);
            rts = __builtin_amdgcn_readlane(rts, src);
            const int s0 = __builtin_amdgcn_readlane(sincl - sl, src);
            it.tiles = (tiles_within(a, it.len) + it.n - 1) / it.n; // chunks of the same length
            const int H = a.cache.numHeads, m = MERGE ? 1 : it.n;
            it.c = k % m;
            it.h = (k / m) % H;
            it.rt = rts - 1 - k / (m * H);
            it.slot = it.n > 1 ? s0 + (k / m) * it.n : -1;
            // offsets that decrease: requests share rows, there may be nothing to work in, and the sum may have passed 2^31
            if (it.n > 1 && (it.slot < 0 || it.slot > s.maxSlots - it.n)) return false;
            return true;
        }
        base = __builtin_amdgcn_readlane(incl, 63);
        sbase = __builtin_amdgcn_readlane(sincl, 63);
    }
    return false;
}

// four adjacent elements of a result (any alignment)
__device__ __forceinline__ void store4(unsigned short* p, f32x4 x, int type) {
    unsigned short r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        r[e] = type == DT_F16 ? __builtin_bit_cast(unsigned short, (_Float16)x[e]) : __builtin_bit_cast(unsigned short, (__bf16)x[e]);
    __builtin_memcpy(p, r, 8);
}

// ---- parts of the two kernels.  A wavefront has NT tiles of 16 rows; lane (n16, grp) = (lane % 16, lane / 16) holds of the scores of
// row n16 of each tile the tokens 16 grp ... + 15 of a step's 64, and of its sums 4 dimensions of every 16.
template <int NT, int MD>
struct Rows {
    float qs[NT];    // what a score is multiplied by beside the block's scale, in units of log 2; not negative
    int limit[NT];   // tokens the row sees
    float top[NT];   // reference of the exponents, log2 of a probability times its value's scale
    float lref[NT];  // reference of the sum of the probabilities: never more than the largest score met so far
    float l[NT];     // sum of the probabilities, in units of 2^(lref - kBias + kRoom)
    float unit[NT];  // one of 2^(top - vref - kBias) in these units
    float vref;      // log2 of the largest value scale met so far
    float base[NT];  // what scores and references are counted from: 0 but where the scores are far from it
    bool far;        // some row's base is not 0
    f32x4 o[NT][MD]; // sums of probability times value, in units of 2^(top - kBias)
    __device__ __forceinline__ void reset() {
        vref = kNoScale;
        far = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            base[t] = 0.f;
            top[t] = lref[t] = kNothing;
            l[t] = unit[t] = 0.f;
#pragma unroll
            for (int i = 0; i < MD; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
};

// NT tiles of rows from row0 on as fp16 operands.  KEYBYTES: step k's dimensions are the ones of the bytes that a lane of the direct
// kernel loads of a key, 64 (k / 2) + 16 grp + 8 (k % 2) ...; else 32 k + 8 grp ...
template <int D, int NT, bool KEYBYTES, int MD>
__device__ __forceinline__ void load_queries(const AttendArgs& a, const Item& it, int G, int row0, int rowsAll, half8_t (&q)[NT][D / 32], Rows<NT, MD>& w) {
    const int lane = threadIdx.x & 63, n16 = lane & 15, grp = lane >> 4;
    constexpr int KS = D / 32;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + n16;
        const bool in = r < rowsAll;
        const int qi = in ? r / G : 0, g = in ? r - qi * G : 0;
        w.limit[t] = !in ? 0 : a.causal ? max(0, it.len - it.nq + qi + 1) : it.len;
        const int64_t at = (int64_t)(it.q0 + qi) * a.qTokenStride + (int64_t)(it.h * G + g) * a.qHeadStride;
        float x[KS][8];
        float big = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d = !KEYBYTES || (D % 64 && k == KS - 1) ? 32 * k + 8 * grp : 64 * (k >> 1) + 16 * grp + 8 * (k & 1);
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
        w.qs[t] = fabsf(a.scale) * kLog2e;
        if (a.type == DT_BF16) {
            big = groups_max(big);
            // largest element to [2^9, 2^10); both factors stay finite: the exponent of a bf16 number is -133 ... 127
            const int e = big > 0.f ? min(max(10 - (int)__builtin_amdgcn_frexp_expf(big), -120), 120) : 0;
            up = __builtin_ldexpf(1.f, e);
            w.qs[t] *= __builtin_ldexpf(1.f, -e);
        }
        if (a.scale < 0.f) up = -up;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[t][k][e] = (_Float16)(x[k][e] * up);
    }
}

// The scores of 64 tokens become probabilities, fp16 operands of the second product; maxima, sums and accumulators follow.
// tok0: the lane group's first token; edge: some row does not see all 64; ks, lvs: the key scale and log2 of the value scale of the
// lane group's block.  A value's scale goes into its probability's exponent, so the sum of the probabilities themselves is the
// lane's sum times the inverse of its scale.  That sum has a reference of its own, the largest top - vref so far: a larger scale
// that comes later takes the row's reference along, and the scores' largest may then lie any distance above top - vref.  No score
// is more than 100 above it (a scale counts as no less than 2^-100 of vref) and the largest is not below it: a step adds no more
// than 2^(14 + 100 - kRoom) per token, and the sum is no less than 2^(kBias - kRoom).  All row tiles are worked on between the same branches: they are independent chains.
// nan: which of the lane group's 16 tokens have a value of code NaN that was taken out (with edge only): rows that see one are NaN.
template <int NT, int MD>
__device__ __forceinline__ void softmax_step(f32x4 (&sc)[NT][4], float ks, float lvs, int tok0, bool edge, unsigned nan, Rows<NT, MD>& w, half8_t (&pr)[NT][2]) {
    float f[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) f[t] = ks * w.qs[t];
    if (edge) {
        if (__ballot(nan != 0)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[t][i][e] = (nan >> (4 * i + e)) & 1 ? __builtin_nanf("") : sc[t][i][e];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][i][e] = (tok0 + 4 * i + e) < w.limit[t] ? sc[t][i][e] * f[t] : -INFINITY;
            f[t] = 1.f;
        }
    }
    if (w.far) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][i][e] = sc[t][i][e] * f[t] - w.base[t]; // (two roundings: the base is such a product)
            f[t] = 1.f;
        }
    }
    const float vnew = fmaxf(w.vref, groups_max(lvs));
    // the exponent of the lane's value scale: where there is none the probability is needed for the sum alone, and is not to raise
    // the reference above the products that count
    const float lv = fmaxf(lvs, vnew - 100.f), iv = __builtin_amdgcn_exp2f(vnew - lv);
    auto lane_max = [&](int t) {
        float mx = highest(sc[t][0][0], sc[t][0][1]);
#pragma unroll
        for (int i = 2; i < 16; ++i) mx = highest(mx, sc[t][i >> 2][i & 3]);
        return mx * f[t];
    };
    auto reference = [&](int t) {
        const float mx = lane_max(t);
        // (2^-22: not below the exact products and sums of the fma below)
        const float all = groups_max(__builtin_fmaf(fabsf(mx), 0x1p-22f, mx) + lv); // (NaN where a group's scores are all masked: passed over)
        // the reference follows the maximum only when that has grown by more than 2^8.  It is that of probability and scale
        // together: what a probability loses in fp16 is then small beside the row's largest term, whatever the scales
        return all > w.top[t] + kSlack ? all : w.top[t];
    };
    float now[NT];
    bool change = vnew != w.vref;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        now[t] = reference(t);
        change |= now[t] != w.top[t];
    }
    if (__ballot(change)) {
        // A reference stands up to 2^-22 of itself above the largest score: the probabilities lose bits from 2^16 on and are zero from
        // 2^27 on.  Such a row's scores are counted from their largest so far instead, as numbers of fp32
        bool far = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) far |= now[t] != w.top[t] && fabsf(now[t]) > kFar && fabsf(now[t]) < INFINITY;
        if (__ballot(far)) {
            w.far = true;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float most = groups_max(lane_max(t));
                const bool moves = now[t] != w.top[t] && fabsf(now[t]) > kFar && fabsf(most) < INFINITY;
                const float by = moves ? most : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[t][i][e] = sc[t][i][e] * f[t] - by;
                f[t] = 1.f;
                w.base[t] += by;
                if (w.top[t] != kNothing) {
                    w.top[t] -= by;
                    w.lref[t] -= by;
                }
                now[t] = reference(t);
            }
        }
        w.vref = vnew;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float od = __builtin_amdgcn_exp2f(w.top[t] - now[t]), ref = fmaxf(w.lref[t], now[t] - vnew);
            w.l[t] *= __builtin_amdgcn_exp2f(w.lref[t] - ref);
            w.unit[t] = __builtin_amdgcn_exp2f((now[t] - vnew) - ref - kRoom);
            w.lref[t] = ref;
            w.top[t] = now[t];
#pragma unroll
            for (int i = 0; i < MD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.o[t][i][e] *= od;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float sub = lv - (w.top[t] - kBias);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i][e], f[t], sub));
                sum += p;
                pr[t][i >> 1][4 * (i & 1) + e] = (_Float16)p;
            }
        w.l[t] = __builtin_fmaf(sum, iv * w.unit[t], w.l[t]);
    }
}

// blocks and scales of a stretch of the context, looked up once: a wait for a block's number in the loop would be a wait for all
// loads issued before it
struct Stretch {
    unsigned at[4 * kSeg]; // where the block's codes of this head begin, in 512 bytes (a block has a multiple of them)
    float ks[4 * kSeg], lvs[4 * kSeg]; // key scale, log2 of the value scale (kNoScale: the values count as zero)
};
__device__ __forceinline__ void look_up(const AttendArgs& a, const Item& it, int seg0, int endAll, int threads, Stretch& z) {
    const int bs = a.cache.blockSize, shift = 31 - __builtin_clz(bs);
    const int* tb = a.table + (int64_t)it.b * a.tableStride;
    for (int i = threadIdx.x; i < 4 * min(kSeg, endAll - seg0); i += threads) {
        const int u = 4 * seg0 + i; // 16 tokens
        int p = -1;
        float ks = 0.f, vs = 0.f;
        if (u < (int)(((unsigned)it.len + 15) >> 4)) { // there should be a block
            const int col = (u << 4) >> shift;
            p = col < a.cols ? tb[col] : -1;
            if ((unsigned)p < (unsigned)a.cache.numBlocks) {
                ks = a.cache.ks[(int64_t)p * a.cache.numHeads + it.h];
                vs = a.cache.vs[(int64_t)p * a.cache.numHeads + it.h];
                // a scale that is negative, infinite or no number makes the scores NaN: the rows that
                // see the block become NaN, those that mask it do not
                if (!(ks >= 0.f && ks < INFINITY && vs >= 0.f && vs < INFINITY)) ks = __builtin_nanf("");
            } else {
                p = -1;
                ks = __builtin_nanf("");
            }
        }
        z.at[i] = (unsigned)((((int64_t)max(p, 0) * a.cache.numHeads + it.h) * (bs * a.cache.headDim)) >> 9);
        z.ks[i] = ks;
        const bool tiny = vs < FLT_MIN; // (the instruction takes subnormal numbers for zero)
        z.lvs[i] = vs > 0.f && vs < INFINITY ? __builtin_amdgcn_logf(tiny ? vs * 0x1p32f : vs) - (tiny ? 32.f : 0.f) : kNoScale;
    }
}

// tokens that a row sees
__device__ __forceinline__ int visible(const AttendArgs& a, const Item& it, int G, int row) {
    return a.causal ? max(0, it.len - it.nq + row / G + 1) : it.len;
}
// the bytes of 16 tokens that lie before the request's end: behind it there may be anything, NaN codes too
__device__ __forceinline__ u32x4 cut_tokens(u32x4 w, int valid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int nb = min(max(valid - 4 * i, 0), 4);
        w[i] &= nb == 4 ? ~0u : (1u << (8 * nb)) - 1u;
    }
    return w;
}
// The 16 tokens of a word quadruple with a NaN code (e4m3 0x7f, 0xff), which are taken out.  Zero times NaN is NaN: a value of
// that code would reach the rows that mask its token too.
template <int CODE>
__device__ __forceinline__ unsigned take_nan(u32x4& w) {
    unsigned m = 0;
    if constexpr (CODE == CACHE_E4M3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned f = ((w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            m |= ((f >> 7 & 1u) | (f >> 14 & 2u) | (f >> 21 & 4u) | (f >> 28 & 8u)) << (4 * i);
            w[i] &= ~((f >> 7) * 0xffu);
        }
    }
    return m;
}
// The sums of the lane groups together.  A NaN code of a value has reached the accumulators of its dimension, or the scores where some
// rows mask it: either way the row is NaN as a whole, its sum too, and so is what it is joined with
template <int NT, int MD>
__device__ __forceinline__ void close_rows(Rows<NT, MD>& w) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float m = w.o[t][0][0];
#pragma unroll
        for (int i = 1; i < 4 * MD; ++i) m = highest(m, w.o[t][i >> 2][i & 3]);
        w.l[t] = groups_sum(w.l[t] + (m - m)); // (sums are finite or NaN)
    }
}
__device__ __forceinline__ float log_sum(float base, float ref, float l) {
    const float up = l < 1.f ? kRoom - kBias : 0.f; // (the two would cancel)
    return l == 0.f ? -INFINITY : (base + (ref + (kRoom - kBias - up) + __builtin_amdgcn_logf(__builtin_ldexpf(l, (int)up)))) * kLn2;
}
// What a row's accumulators are multiplied by to become its result, as a factor and a power of two: the scales of the values go up
// to the largest fp32 numbers and the sums beyond them, the results do not
struct Norm {
    float f;
    int e;
    __device__ __forceinline__ Norm(float top, float lref, float l) {
        const float x = top - lref - kRoom, whole = floorf(x);
        f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(x - whole) / l;
        e = l == 0.f ? 0 : (int)whole;
    }
    __device__ __forceinline__ f32x4 operator()(f32x4 x) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_ldexpf(x[i] * f, e);
        return x;
    }
};
// Partial results (of a wavefront, of a chunk) are results of their own tokens, with the reference and the sum of their
// probabilities: they are joined with weights that add up to one.  Where a part saw nothing its sum and result are zero.
struct Part {
    float base, ref, l;
    __device__ __forceinline__ float above(const Part& o) const { return (base - o.base) + (ref - o.ref); } // of references
    __device__ __forceinline__ void raise(const Part& o) { // to the larger reference
        const bool up = o.above(*this) > 0.f;
        base = up ? o.base : base;
        ref = up ? o.ref : ref;
    }
    __device__ __forceinline__ float weight(const Part& most) const { return l * __builtin_amdgcn_exp2f(above(most)); }
};
// A sum of zero is that of a row that sees nothing, or of one all of whose scores are -inf (an infinite query): that one is NaN
__device__ __forceinline__ float sum_seen(float l, int sees) { return l == 0.f && sees > 0 ? __builtin_nanf("") : l; }
// a row of a wavefront's own: the result, or a chunk's partial sums
template <int D, int NT, int MD>
__device__ __forceinline__ void write_rows(const AttendArgs& a, const Sched& s, const Item& it, int G, int row0, int rowsAll, Rows<NT, MD>& w) {
    const int lane = threadIdx.x & 63, n16 = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 16 * t + n16;
        if (r >= rowsAll) continue;
        if (it.slot < 0) w.l[t] = sum_seen(w.l[t], visible(a, it, G, r));
        const Norm norm(w.top[t], w.lref[t], w.l[t]);
        if (it.slot >= 0) {
            const int64_t pr = (int64_t)(it.slot + it.c) * s.rows + (r - it.rt * s.rows);
#pragma unroll
            for (int i = 0; i < MD; ++i) *(f32x4*)(s.partO + pr * D + 16 * i + 4 * grp) = norm(w.o[t][i]);
            if (grp == 0) s.partML[pr] = make_float4(w.base[t], w.lref[t], w.l[t], 0.f);
        } else {
            const int qi = r / G, g = r - qi * G;
            unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + 4 * grp;
#pragma unroll
            for (int i = 0; i < MD; ++i) store4(op + 16 * i, norm(w.o[t][i]), a.type);
            if (grp == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = log_sum(w.base[t], w.lref[t], w.l[t]);
        }
    }
}

// Few rows (single tokens, drafts): bound by the bytes of the cache.  The four wavefronts of a workgroup share the rows and take every
// fourth tile of the chunk, straight from memory into the registers that feed the matrix instructions; their results are joined in
// LDS.  A tile's values are asked for before its scores are computed and the next tile's keys before its softmax; what a wait would
// hold up is looked up beforehand (Stretch).
// 64 ragged contexts of up to 16384 tokens, 8 heads of 128, e4m3 (1.34 GB): 263 us, 5.1 TB/s, as fast as a large copy; 3 of 131071,
// one head of 256, int8 (0.2 GB): 50 us, 4.0 TB/s (367 registers: one wavefront per SIMD); 1 of 1000: 12 us, a chain of dependent
// loads (lengths, blocks, scales, keys, values).  Drafts over the ragged contexts, 2 / 4 / 5 / 8 queries each, 4 heads to one: 259 / 268 / 277 /
// 284 us a call (one: 252).
template <int D, int CODE, int NT>
__global__ __launch_bounds__(256) void cache_attend_direct_kernel(AttendArgs a, Sched s) {
    constexpr int KS = D / 32, MD = D / 16; // steps of the first product, row tiles of the second
    constexpr int NL = D / 64;              // 16-byte pieces of a key per lane (and one of 8 bytes if D % 64)
    constexpr int ROWS = 16 * NT;
    Item it;
    if (!find_item<false>(a, s, blockIdx.x, it)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n16 = lane & 15, grp = lane >> 4;
    const int H = a.cache.numHeads, G = a.heads / H, bs = a.cache.blockSize;
    const int rowsAll = it.nq * G, row0 = it.rt * ROWS;
    const int vis = visible(a, it, G, min(rowsAll, row0 + ROWS) - 1), visMin = visible(a, it, G, row0); // what the last / the first row sees
    const int tile0 = it.c * it.tiles, end = min(tile0 + it.tiles, tiles_of(vis));
    int tile = tile0 + wave;
    __shared__ Stretch z;

    // the codes of a tile, on their way or there
    u32x4 kr[4][NL];
    u32x2 kx[4];
    u32x4 vr[MD];
    auto fetch_k = [&](int t, unsigned at) {
        const int off = ((t * kTile + 16 * (n16 >> 2)) & (bs - 1)) + (n16 & 3);
        const uint8_t* p = a.cache.k + ((uint64_t)at << 9) + off * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < NL; ++j) kr[i][j] = *(const u32x4*)(p + i * 4 * D + 64 * j + 16 * grp);
            if constexpr (D % 64) kx[i] = *(const u32x2*)(p + i * 4 * D + 64 * NL + 8 * grp);
        }
    };
    auto fetch_v = [&](int t, unsigned at) { // 16 tokens of a dimension per lane
        const uint8_t* p = a.cache.v + ((uint64_t)at << 9) + n16 * bs + ((t * kTile + 16 * grp) & (bs - 1));
#pragma unroll
        for (int i = 0; i < MD; ++i) vr[i] = *(const u32x4*)(p + i * 16 * bs);
    };
    // the first keys are on their way before the queries are looked at
    look_up(a, it, tile0, end, 256, z);
    __syncthreads();
    if (tile < min(tile0 + kSeg, end)) fetch_k(tile, z.at[(tile - tile0) * 4 + (n16 >> 2)]);
    half8_t q[NT][KS];
    Rows<NT, MD> w;
    load_queries<D, NT, true>(a, it, G, row0, rowsAll, q, w);
    w.reset();

    for (int seg0 = tile0; seg0 < end; seg0 += kSeg) {
        const int segEnd = min(seg0 + kSeg, end);
        if (seg0 != tile0) {
            __syncthreads(); // (the stretch before has been read)
            look_up(a, it, seg0, end, 256, z);
            __syncthreads();
            if (tile < segEnd) fetch_k(tile, z.at[(tile - seg0) * 4 + (n16 >> 2)]);
        }
        for (; tile < segEnd; tile += kWaves) {
            const int t0 = tile * kTile, u = (tile - seg0) * 4;
            fetch_v(tile, z.at[u + grp]);
            const float ks = z.ks[u + grp], lvs = z.lvs[u + grp];
            f32x4 sc[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    u32x2 c;
                    if ((D % 64) && k == KS - 1)
                        c = kx[i];
                    else
                        c = (k & 1) ? u32x2{kr[i][k >> 1][2], kr[i][k >> 1][3]} : u32x2{kr[i][k >> 1][0], kr[i][k >> 1][1]};
                    const half8_t ka = widen<CODE>(c);
#pragma unroll
                    for (int t = 0; t < NT; ++t) sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, q[t][k], sc[t][i], 0, 0, 0);
                }
            }
            if (tile + kWaves < segEnd) fetch_k(tile + kWaves, z.at[u + 4 * kWaves + (n16 >> 2)]);
            half8_t pr[NT][2];
            unsigned nan = 0;
            if (CODE == CACHE_E4M3 && visMin < it.len && t0 + kTile > visMin) { // some rows mask tokens that others see
#pragma unroll
                for (int i = 0; i < MD; ++i) nan |= take_nan<CODE>(vr[i]);
#pragma unroll
                for (int o = 8; o; o >>= 1) nan |= (unsigned)__shfl_xor((int)nan, o, 64);
                if (lvs == kNoScale) nan = 0; // (cut below: zero whatever the codes)
            }
            softmax_step(sc, ks, lvs, t0 + 16 * grp, t0 + kTile > visMin, nan, w, pr);
            if (t0 + kTile > it.len || __ballot(lvs == kNoScale)) {
#pragma unroll
                for (int i = 0; i < MD; ++i) vr[i] = cut_tokens(vr[i], lvs == kNoScale ? 0 : it.len - (t0 + 16 * grp));
            }
#pragma unroll
            for (int i = 0; i < MD; ++i) {
                const half8_t a0 = widen<CODE>(u32x2{vr[i][0], vr[i][1]}), a1 = widen<CODE>(u32x2{vr[i][2], vr[i][3]});
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    w.o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pr[t][0], w.o[t][i], 0, 0, 0);
                    w.o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pr[t][1], w.o[t][i], 0, 0, 0);
                }
            }
        }
    }
    close_rows(w);

    constexpr int PITCH = D + 4;
    __shared__ __align__(16) float sm[kWaves][16 * NT][PITCH];
    __shared__ Part sml[kWaves][16 * NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (grp == 0) sml[wave][16 * t + n16] = {w.base[t], w.lref[t], w.l[t]};
        const Norm norm(w.top[t], w.lref[t], w.l[t]);
#pragma unroll
        for (int i = 0; i < MD; ++i) *(f32x4*)&sm[wave][16 * t + n16][16 * i + 4 * grp] = norm(w.o[t][i]);
    }
    __syncthreads();
    // a thread joins 4 dimensions of a row
    for (int x = threadIdx.x; x < 16 * NT * (D / 4); x += 256) {
        const int r = x / (D / 4), d = 4 * (x - r * (D / 4));
        if (row0 + r >= rowsAll) break;
        Part M = sml[0][r];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) M.raise(sml[v][r]);
        float L = 0.f, wt[kWaves];
#pragma unroll
        for (int v = 0; v < kWaves; ++v) L += wt[v] = sml[v][r].weight(M);
        if (it.slot < 0) L = sum_seen(L, visible(a, it, G, row0 + r));
        const float inv = L == 0.f ? 0.f : 1.f / L;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const float f = wt[v] * inv;
            const f32x4 ow = *(const f32x4*)&sm[v][r][d];
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = __builtin_fmaf(f, ow[e], O[e]);
        }
        if (it.slot >= 0) {
            const int64_t pr = (int64_t)(it.slot + it.c) * ROWS + r;
            *(f32x4*)(s.partO + pr * D + d) = O;
            if (d == 0) s.partML[pr] = make_float4(M.base, M.ref, L, 0.f);
        } else {
            const int qi = (row0 + r) / G, g = (row0 + r) - qi * G;
            unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + d;
            store4(op, O, a.type);
            if (d == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = log_sum(M.base, M.ref, L);
        }
    }
}

// Many rows (prompts): bound by the arithmetic.  Each of the WAVES wavefronts has rows of its own; a tile's keys and values are loaded
// and widened to fp16 once for all of them and laid into LDS fragment by fragment, in the order in which the matrix instructions'
// lanes read them (no bank conflicts on either side).  Two such buffers: the next tile is loaded while one is worked on.
// Four requests of 2048 queries that end at token 8195, 16 heads over 4 of 128, e4m3: the call takes 563 - 569 us, 850 TFLOP/s.  The matrix
// pipe is busy 35 % of the time: beside 64 matrix instructions a wavefront issues 265 other vector instructions per tile (34 of them
// transcendental), and 250 registers leave two wavefronts per SIMD.  Half of the wavefronts half a tile behind the others (before the last
// steps, which took 595 to 574) 620; the next tile's products between the softmax's instructions: it spills.  Ragged prompts: 356 us, of which
// the longest work item alone takes some 330 (256 rows that see 8192 tokens, at what a CU does here); straight from memory, as above, 745.
template <int D, int CODE, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void cache_attend_rows_kernel(AttendArgs a, Sched s) {
    constexpr int KS = D / 32, MD = D / 16;
    constexpr int ROWS = 16 * NT * WAVES;
    constexpr int KP = 4 * ((D + 63) / 64);              // pieces of the keys: 16 tokens x 64 dimensions, a wavefront each
    constexpr int KW = (KP + WAVES - 1) / WAVES, VW = (MD + WAVES - 1) / WAVES;
    Item it;
    if (!find_item<false>(a, s, blockIdx.x, it)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n16 = lane & 15, grp = lane >> 4;
    const int H = a.cache.numHeads, G = a.heads / H, bs = a.cache.blockSize;
    const int rowsAll = it.nq * G, row0 = it.rt * ROWS + wave * 16 * NT;
    const int lastRow = min(rowsAll, row0 + 16 * NT) - 1;
    const int vis = lastRow >= row0 ? visible(a, it, G, lastRow) : 0, visMin = lastRow >= row0 ? visible(a, it, G, row0) : 0;
    const int tile0 = it.c * it.tiles;
    const int end = min(tile0 + it.tiles, tiles_of(vis));
    const int endAll = min(tile0 + it.tiles, tiles_of(visible(a, it, G, min(rowsAll, it.rt * ROWS + ROWS) - 1)));
    __shared__ Stretch z;
    __shared__ __align__(16) half8_t kf[2][4 * KS][64]; // fragment (i, k): tokens 16 g + 4 i + e in row 4 g + e, dimensions 32 k ...
    __shared__ __align__(16) half8_t vf[2][MD * 2][64]; // fragment (i, h): dimensions 16 i ..., tokens 16 grp + 8 h ...

    __shared__ unsigned nanL[3][4]; // tokens with NaN codes of a tile's four groups; of this tile, the next, and one being cleared
    const int visMinAll = visible(a, it, G, it.rt * ROWS);

    u32x4 kr[KW], vr[VW];
    // (every wavefront loads, also where there is nothing for it: a load under a condition waits for the loads before it)
    auto fetch = [&](int t, int seg0) {
        const int u = (t - seg0) * 4;
        const uint8_t* k = a.cache.k + ((uint64_t)z.at[u + (n16 >> 2)] << 9) + (((t * kTile + 16 * (n16 >> 2)) & (bs - 1)) + (n16 & 3)) * D;
        const uint8_t* v = a.cache.v + ((uint64_t)z.at[u + grp] << 9) + n16 * bs + ((t * kTile + 16 * grp) & (bs - 1));
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const int pc = min(wave + j * WAVES, KP - 1);
            kr[j] = *(const u32x4*)(k + 4 * (pc & 3) * D + min(64 * (pc >> 2) + 16 * grp, D - 16));
        }
#pragma unroll
        for (int j = 0; j < VW; ++j) vr[j] = *(const u32x4*)(v + 16 * min(wave + j * WAVES, MD - 1) * bs);
    };
    auto lay = [&](int t, int seg0, int buf) { // what fetch brought
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            const int pc = wave + j * WAVES, i = pc & 3, d = 64 * (pc >> 2) + 16 * grp;
            if (pc < KP && d < D) {
                kf[buf][i * KS + d / 32][((d >> 3) & 3) * 16 + n16] = widen<CODE>(u32x2{kr[j][0], kr[j][1]});
                kf[buf][i * KS + d / 32][(((d >> 3) & 3) + 1) * 16 + n16] = widen<CODE>(u32x2{kr[j][2], kr[j][3]});
            }
        }
        const bool none = z.lvs[(t - seg0) * 4 + grp] == kNoScale, tail = (t + 1) * kTile > it.len || __ballot(none);
        const int valid = none ? 0 : it.len - (t * kTile + 16 * grp);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const int i = wave + j * WAVES;
            if (i < MD) {
                u32x4 c = vr[j];
                if (tail) { // (a branch: as a selection it costs 39 instructions in every tile)
                    asm volatile("");
                    c = cut_tokens(c, valid);
                }
                if (CODE == CACHE_E4M3 && visMinAll < it.len && (t + 1) * kTile > visMinAll) { // some rows mask tokens that others see
                    const unsigned nan = take_nan<CODE>(c);
                    if (nan) atomicOr(&nanL[t % 3][grp], nan);
                }
                vf[buf][2 * i][lane] = widen<CODE>(u32x2{c[0], c[1]});
                vf[buf][2 * i + 1][lane] = widen<CODE>(u32x2{c[2], c[3]});
            }
        }
    };
    half8_t q[NT][KS];
    Rows<NT, MD> w;
    load_queries<D, NT, false>(a, it, G, row0, rowsAll, q, w);
    w.reset();
    for (int seg0 = tile0; seg0 < endAll; seg0 += kSeg) {
        const int segEnd = min(seg0 + kSeg, endAll);
        __syncthreads(); // (the stretch before has been read)
        look_up(a, it, seg0, endAll, 64 * WAVES, z);
        if (threadIdx.x < 12) nanL[threadIdx.x >> 2][threadIdx.x & 3] = 0;
        __syncthreads();
        fetch(seg0, seg0);
        lay(seg0, seg0, seg0 & 1);
        __syncthreads();
        for (int tile = seg0; tile < segEnd; ++tile) {
            const int buf = tile & 1, t0 = tile * kTile, u = (tile - seg0) * 4;
            const bool more = tile + 1 < segEnd;
            fetch(min(tile + 1, segEnd - 1), seg0);
            if (threadIdx.x < 4) nanL[(tile + 2) % 3][threadIdx.x] = 0;
            if (tile < end) {
                const float ks = z.ks[u + grp], lvs = z.lvs[u + grp];
                f32x4 sc[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                // four fragments at a time, the next four on their way from LDS; the order is pinned, or the compiler waits for
                // each one right before its use
                half8_t fr[2][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) fr[0][j] = kf[buf][j][lane];
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                for (int g = 0; g < KS; ++g) {
                    if (g + 1 < KS) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) fr[(g + 1) & 1][j] = kf[buf][4 * (g + 1) + j][lane];
                        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = (4 * g + j) / KS, k = (4 * g + j) % KS;
#pragma unroll
                        for (int t = 0; t < NT; ++t) sc[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[g & 1][j], q[t][k], sc[t][i], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x8, 4 * NT, 0);
                }
                half8_t pr[NT][2];
                // (lay took the codes out wherever some row of the workgroup masks part of the tile: the wavefronts that see all of
                // it get them back too)
                unsigned nan = 0;
                if (CODE == CACHE_E4M3 && visMinAll < it.len && t0 + kTile > visMinAll) nan = nanL[tile % 3][grp];
                softmax_step(sc, ks, lvs, t0 + 16 * grp, t0 + kTile > visMin || __ballot(nan != 0), nan, w, pr);
#pragma unroll
                for (int j = 0; j < 4; ++j) fr[0][j] = vf[buf][j][lane];
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
                for (int g = 0; g < MD / 2; ++g) {
                    if (g + 1 < MD / 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) fr[(g + 1) & 1][j] = vf[buf][4 * (g + 1) + j][lane];
                        __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                w.o[t][2 * g + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fr[g & 1][2 * j + h], pr[t][h], w.o[t][2 * g + j], 0, 0, 0);
                    __builtin_amdgcn_sched_group_barrier(0x8, 4 * NT, 1);
                }
            }
            if (more) lay(tile + 1, seg0, buf ^ 1);
            __syncthreads();
        }
    }
    close_rows(w);
    write_rows<D>(a, s, it, G, row0, rowsAll, w);
}

// Joins the chunks of a split request: a workgroup takes every mergeRows-th row.  The chunks' weights come first (all loads in flight together), then
// every group of dim / 4 threads adds up its share of the chunks, eight loads at a time.
constexpr int kMergeChunks = 1024; // weights held at once
__global__ __launch_bounds__(256) void cache_attend_merge_kernel(AttendArgs a, Sched s) {
    Item it;
    if (!find_item<true>(a, s, blockIdx.x / s.mergeRows, it)) return;
    const int D = a.cache.headDim, G = a.heads / a.cache.numHeads;
    const int quads = D / 4, parts = 256 / quads;
    const int part = threadIdx.x / quads, d = 4 * (threadIdx.x - part * quads);
    if (it.n <= 8) { // few chunks: every group of threads joins a row of its own
        if (part >= parts) return;
        for (int r = (blockIdx.x % s.mergeRows) * parts + part; r < s.rows; r += s.mergeRows * parts) {
            const int row = it.rt * s.rows + r;
            if (row >= it.nq * G) return;
            const int64_t at = (int64_t)it.slot * s.rows + r;
            Part x[8];
            f32x4 v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int64_t p = at + (int64_t)min(c, it.n - 1) * s.rows;
                const float4 ml = s.partML[p];
                x[c] = {ml.x, ml.y, ml.z};
                v[c] = *(const f32x4*)(s.partO + p * D + d);
            }
            Part M = x[0];
#pragma unroll
            for (int c = 1; c < 8; ++c) M.raise(x[c]); // (those behind the last are the last)
            float L = 0.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) L += x[c].l = c < it.n ? x[c].weight(M) : 0.f;
            L = sum_seen(L, visible(a, it, G, row));
            const float inv = L == 0.f ? 0.f : 1.f / L;
            f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) O[j] = __builtin_fmaf(x[c].l * inv, v[c][j], O[j]);
            const int qi = row / G, g = row - qi * G;
            unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + d;
            store4(op, O, a.type);
            if (d == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = log_sum(M.base, M.ref, L);
        }
        return;
    }
    __shared__ __align__(16) float so[256 * 4];
    __shared__ float wt[kMergeChunks];
    __shared__ Part redM[4];
    __shared__ float red[4];
    for (int r = blockIdx.x % s.mergeRows; r < s.rows; r += s.mergeRows) {
        const int row = it.rt * s.rows + r;
        if (row >= it.nq * G) return;
        __syncthreads(); // (the row before has been joined)
        const float4* ml = s.partML + (int64_t)it.slot * s.rows + r;
        auto part_of = [&](int c) {
            const float4 x = ml[(int64_t)c * s.rows];
            return Part{x.x, x.y, x.z};
        };
        const float* po = s.partO + ((int64_t)it.slot * s.rows + r) * D;
        const Part mine = part_of(min((int)threadIdx.x, it.n - 1)); // (one chunk a thread is what there mostly is)
        Part M = mine;
        for (int c = threadIdx.x + 256; c < it.n; c += 256) M.raise(part_of(c));
#pragma unroll
        for (int o = 32; o; o >>= 1) M.raise({__shfl_xor(M.base, o, 64), __shfl_xor(M.ref, o, 64), 0.f});
        if ((threadIdx.x & 63) == 0) redM[threadIdx.x >> 6] = M;
        __syncthreads();
        M = redM[0];
        for (int v = 1; v < 4; ++v) M.raise(redM[v]);
        float L = 0.f;
        for (int c = threadIdx.x; c < it.n; c += 256) {
            const float f = (c == (int)threadIdx.x ? mine : part_of(c)).weight(M);
            if (c < kMergeChunks) wt[c] = f;
            L += f;
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = L;
        __syncthreads();
        L = sum_seen(red[0] + red[1] + red[2] + red[3], visible(a, it, G, row));
        const float inv = L == 0.f ? 0.f : 1.f / L;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < it.n; c0 += kMergeChunks) {
            const int n = min(it.n - c0, kMergeChunks);
            if (c0) {
                __syncthreads();
                for (int c = threadIdx.x; c < n; c += 256) wt[c] = part_of(c0 + c).weight(M);
                __syncthreads();
            }
            if (part < parts) {
                const float* p = po + (int64_t)c0 * s.rows * D + d;
                int c = part;
                for (; c + 7 * parts < n; c += 8 * parts) {
                    f32x4 v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = *(const f32x4*)(p + (int64_t)(c + e * parts) * s.rows * D);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float f = wt[c + e * parts] * inv;
#pragma unroll
                        for (int j = 0; j < 4; ++j) O[j] = __builtin_fmaf(f, v[e][j], O[j]);
                    }
                }
                for (; c < n; c += parts) {
                    const f32x4 v = *(const f32x4*)(p + (int64_t)c * s.rows * D);
                    const float f = wt[c] * inv;
#pragma unroll
                    for (int j = 0; j < 4; ++j) O[j] = __builtin_fmaf(f, v[j], O[j]);
                }
            }
        }
        *(f32x4*)&so[4 * threadIdx.x] = O;
        __syncthreads();
        if (threadIdx.x >= quads) continue;
        for (int p = 1; p < parts; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] += so[4 * (p * quads + threadIdx.x) + e];
        const int qi = row / G, g = row - qi * G;
        unsigned short* op = (unsigned short*)a.out + (int64_t)(it.q0 + qi) * a.outTokenStride + (int64_t)(it.h * G + g) * a.outHeadStride + d;
        store4(op, O, a.type);
        if (d == 0 && a.lse) a.lse[(int64_t)(it.q0 + qi) * a.heads + it.h * G + g] = log_sum(M.base, M.ref, L);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// rows of a work item and the requests it serves
struct Launch {
    Sched s;
    int nt, waves;
    int64_t grid, mergeGrid;
    size_t bytes;
};

int plan_launches(const AttendArgs& a, int num_cus, Launch out[2]) {
    const int G = a.heads / a.cache.numHeads, D = a.cache.headDim;
    const int64_t most = (int64_t)a.maxQueries * G;
    int n = 0;
    auto add = [&](int nt, int waves, int lo, int64_t hi) { // waves 0: the direct kernel
        Launch& L = out[n++];
        L.nt = nt;
        L.waves = waves;
        Sched& s = L.s;
        s.rows = 16 * nt * (waves ? waves : 1);
        s.rowShift = 0;
        while ((1 << s.rowShift) < s.rows) ++s.rowShift;
        s.rowLo = lo;
        s.rowHi = (int)std::min<int64_t>(hi, INT32_MAX);
        // Direct: twice as many chunks as there are workgroups at work at a time, one and a half times with one workgroup on a CU
        // (131071 tokens, 256 dimensions: 256 / 384 / 512 / 768 chunks 57 / 48 / 56 / 57 us)
        s.target = waves ? num_cus * 8 / waves : num_cus * (D <= 64 ? 12 : D <= 128 ? 8 : 3) / 2;
        s.slack = waves ? 2 : 1;
        s.sort = waves != 0;
        const int64_t rowTiles = std::min(((int64_t)a.tokens * G + s.rows - 1) / s.rows + a.batch, (int64_t)a.batch * ((s.rowHi + (int64_t)s.rows - 1) / s.rows));
        const int64_t tiles = ((int64_t)a.cols * a.cache.blockSize + kTile) / kTile;
        // a split costs a launch to join it (4 us), a tile of a wavefront 1 us: where the table holds no more than 16 tiles nothing is
        // split.  What the host can go by is the table's width, not the lengths: 1000 tokens take 11.9 us through a table of 63 blocks of
        // 16, 13.3 through one of 512 (split, joined), 50 tokens 7.8 and 9.7 (a join that finds nothing)
        s.minTiles = waves || tiles > 16 ? 8 : 16;
        s.wshift = 0;
        while (((rowTiles * tiles) >> s.wshift) + a.batch > (int64_t)1 << 30) ++s.wshift;
        s.merge = tiles > s.minTiles;
        // a request with n > 1 chunks has at most twice its share of the total in them
        const int64_t items = s.merge ? 2 * (int64_t)s.target + 2 * (int64_t)a.cache.numHeads : 0;
        s.maxSlots = (int)std::min<int64_t>(items, INT32_MAX);
        L.grid = rowTiles * a.cache.numHeads + items;
        const int64_t groups = std::min<int64_t>(rowTiles * a.cache.numHeads, s.maxSlots / 2);
        s.mergeRows = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(s.rows, most), 2048 / std::max<int64_t>(groups, 1)));
        L.mergeGrid = s.merge ? groups * s.mergeRows : 0;
        L.bytes = s.merge ? round_up((size_t)s.maxSlots * s.rows * D * 4, 256) + round_up((size_t)s.maxSlots * s.rows * 16, 256) : 0;
        s.partO = nullptr;
        s.partML = nullptr;
    };
    // 256 dimensions and 32 rows do not fit the registers of a wavefront (nor 192, where two of them share a SIMD)
    const int wide = D > 192 ? 1 : 2;
    // few rows (single tokens, drafts): the wavefronts of a workgroup split the tokens; many rows: they split the rows
    if (most <= 16) {
        add(1, 0, 1, INT64_MAX);
    } else if (most <= 32) {
        add(wide, 0, 1, INT64_MAX);
    } else {
        if (a.queryOffsets && G <= 32) add(G <= 16 ? 1 : wide, 0, 1, G <= 16 ? 16 : 32);
        // 128 rows of a workgroup, two of them on a CU, or 256
        add(D > 128 ? 1 : 2, D > 128 || most > 128 ? 8 : 4, n ? out[0].s.rowHi + 1 : 1, INT64_MAX);
    }
    return n;
}

template <int D, int CODE>
void launch_one(const AttendArgs& a, const Launch& L, hipStream_t stream) {
    const dim3 grid((unsigned)L.grid);
    if (L.waves == 8) {
        cache_attend_rows_kernel<D, CODE, (D > 128 ? 1 : 2), 8><<<grid, 512, 0, stream>>>(a, L.s);
    } else if (L.waves == 4) {
        if constexpr (D <= 128) cache_attend_rows_kernel<D, CODE, 2, 4><<<grid, 256, 0, stream>>>(a, L.s);
    } else if (L.nt == 1) {
        cache_attend_direct_kernel<D, CODE, 1><<<grid, 256, 0, stream>>>(a, L.s);
    } else {
        if constexpr (D <= 192) cache_attend_direct_kernel<D, CODE, 2><<<grid, 256, 0, stream>>>(a, L.s);
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

int64_t cache_attend_threads(const AttendArgs& a) {
    Launch L[2];
    const int n = plan_launches(a, 256, L); // (fewer CUs make fewer)
    int64_t most = 0;
    for (int i = 0; i < n; ++i) most = std::max({most, L[i].grid * (L[i].waves ? 64 * L[i].waves : 256), L[i].mergeGrid * 256});
    return most;
}

void launch_cache_attend(const AttendArgs& a, int num_cus, hipStream_t stream) {
    Launch L[2];
    const int n = plan_launches(a, num_cus, L);
    char* ws = (char*)a.workspace;
    for (int i = 0; i < n; ++i) {
        Sched& s = L[i].s;
        if (s.merge) {
            s.partO = (float*)ws;
            s.partML = (float4*)(ws + round_up((size_t)s.maxSlots * s.rows * a.cache.headDim * 4, 256));
            ws += L[i].bytes;
        }
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
