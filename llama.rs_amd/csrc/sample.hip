// sample.hip — one token of each row of logits from a given random number:
// temperature, top-k, top-p, min-p (Sampler::sample, llama-sampling/src/
// sampler.rs:24-88, does the first three on the host).
//
// The order of a row's words is logit descending, index ascending; weights are
// w_i = e^((l_i - l_max) / T).  The kept set is a prefix of that order:
//   K  the first top_k words (0: all)
//   P  the shortest prefix of K whose weights sum to at least top_p times K's
//   M  the words of P with w >= min_p
// and the token is the least index i of M with sum_{j in M, j <= i} w_j > u S,
// S = sum_M w: the inverse of the distribution function in index order, which
// needs no sorted copy of the row.  NaN counts as -inf and is never taken.
//
// A word is one 64-bit value, ordered as the row is: the logit's bits made
// monotone, then the complement of its index, so that no two are equal and ties
// go to the lower index.  Weights are whole multiples of 2^-42 (of the largest
// word's weight) in 64 bits: their sums do not depend on the order in which
// atomics or wavefronts add them, 2^21 words cannot overflow them, and a sum is
// off by less than 2^-43 per word.  exp is evaluated in double: the cuts and the
// token depend on sums next to a border, where 2^-24 of a sum is many words.
//
// Two forms.  top_k up to TK (greedy rows among them: top_k = 1): each
// workgroup selects the top_k of its part of a row (k_part), one workgroup per
// row merges the parts and picks (k_pick).  Otherwise: the row's range (k_range),
// a histogram of 1024 bins over it (k_hist), the words of the bins in which the
// cuts fall and the sums of the parts above (k_collect), the cuts and the token
// (k_finish).  Up to top_k LIST / 2 the list usually has room for every word from
// the top down to top-k's bin: then no weights are summed by bin, the cuts and the
// token come from the list, and the row itself is read again only where equal
// logits overflow it.
//
// A row is read once by the first form and three times by the second (the second
// and third time out of the caches); below some 10 MB of logits the launches and
// the chains of barriers within them bound both: 9.7 us for a row of 32000 at
// top_k 40, 24 for a row of 152064 at top_p 0.9, 16 for 25 such rows at top_k 50,
// 55 for 64 rows of 248320 at top_k 1000 (13 to read them once).
#include "lrs_internal.h"

namespace lrs {

namespace {

typedef unsigned long long u64;

constexpr uint32_t TK = 128;        // top_k of the first form
constexpr uint32_t PICK_MAX = 8192; // words that a row's parts give it at most
constexpr uint32_t NB = 1024;       // bins of the second form
constexpr uint32_t LIST = 2048;     // words of the cuts' bins kept per row
constexpr uint32_t WG = 1024;       // threads of a workgroup of the second form: a part in one go where there is one row
constexpr uint32_t MAX_PARTS = 256;  // of the first form; 64 of the second, one for each lane
constexpr double ONE = 4398046511104.0;  // 2^42

struct Row {
    const float *x;
    size_t ld;
    uint32_t vocab, parts, part;  // part: words per workgroup (second form)
    double inv_t;
    float top_p, min_p, temp;
    uint32_t k;  // 0: all
    const float *u;
    uint32_t *tok;
    float *prob;           // or null
    uint32_t *step, *gen;  // the token as the next step's too (row 0), or null
    uint32_t gen_cap;
    bool vec;     // rows are 16-byte aligned
    bool listed;  // second form: every word that top-k may keep is in the row's list
};

// the logit as an unsigned number of the same order; 0: never taken
__device__ __forceinline__ uint32_t ord(float l) {
    const float z = l + 0.0f;  // -0 and 0 tie
    if (!(z > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(z);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ u64 word(float l, uint32_t i) {
    const uint32_t k = ord(l);
    return k ? (u64)k << 32 | (0xFFFFFFFFu - i) : 0ull;
}
__device__ __forceinline__ uint32_t word_index(u64 w) { return 0xFFFFFFFFu - (uint32_t)w; }
__device__ __forceinline__ float word_logit(u64 w) { return unord((uint32_t)(w >> 32)); }

// e^x, x <= 0 (0 below -800): e^x = 2^n e^r with |r| <= ln 2 / 2, the series to
// r^11 (r^12 / 12! < 2^-47 of it)
__device__ __forceinline__ double exp_neg(double x) {
    x = fmax(x, -800.0);
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));
    double p = 1.0 / 39916800;
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// e^((l - top) / T), 1 for the top's equals (an infinite top leaves the rest nothing)
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    return l == top ? 1.0 : exp_neg(((double)l - (double)top) * inv_t);
}
// in whole multiples of 2^-42: the sum with 2^52 rounds to one
__device__ __forceinline__ u64 fixed(double w) {
    return (u64)__double_as_longlong(w * ONE + 4503599627370496.0) - 0x4330000000000000ull;
}

// l[0..4) of elements i.. of a row, -inf past its end
__device__ __forceinline__ void load4(const Row &a, const float *x, uint32_t i, float (&l)[4]) {
    if (a.vec && i + 4 <= a.vocab) {
        const float4 v = *reinterpret_cast<const float4 *>(x + i);
        l[0] = v.x, l[1] = v.y, l[2] = v.z, l[3] = v.w;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) l[j] = i + j < a.vocab ? x[i + j] : -INFINITY;
    }
}

// sums over the lanes up to and with each one (DPP moves: a shuffle goes through LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_from(u64 x) {
    return (u64)dpp_from<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | dpp_from<CTRL, ROWS>((uint32_t)x);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
    x += dpp_from<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: rows of sixteen
    x += dpp_from<0x112, 0xf>(x);
    x += dpp_from<0x114, 0xf>(x);
    x += dpp_from<0x118, 0xf>(x);
    x += dpp_from<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    x += dpp_from<0x143, 0xc>(x);
    return x;
}
__device__ __forceinline__ u64 lane_value(u64 x, uint32_t lane) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// the token is the first word at which the running sum (of whole numbers) is
// above this: floor(u sum), below sum itself
__device__ __forceinline__ u64 target(const Row &a, uint32_t row, u64 sum) {
    const float u = a.u[row];
    return u > 0.f ? (u < 1.f ? min((u64)((double)u * (double)sum), sum - 1) : sum - 1) : 0ull;
}

__device__ __forceinline__ void emit(const Row &a, uint32_t row, uint32_t tok, float p) {
    a.tok[row] = tok;
    if (a.prob) a.prob[row] = p;
    if (a.step && row == 0) {
        const uint32_t n = a.step[2];
        if (a.gen && n < a.gen_cap) a.gen[n] = tok;
        a.step[0] = tok;
        a.step[1] = a.step[1] + 1;
        a.step[2] = n + 1;
    }
}

// ---- top_k up to TK -------------------------------------------------------
typedef u64 u64x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// how many of list's words (zeros behind them up to a multiple of 8) are above w;
// the reads of eight words are in flight together
__device__ __forceinline__ uint32_t above(const u64 *list, uint32_t n, u64 w) {
    uint32_t r = 0;
    for (uint32_t j = 0; j < n; j += 8) {
        u64x2 v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = *reinterpret_cast<const u64x2 *>(list + j + 2 * e);
#pragma unroll
        for (int e = 0; e < 4; e++) r += (v[e][0] > w) + (v[e][1] > w);
    }
    return r;
}

// The top_k words of a part (a.part words, at most 1024 E): word j of part g in
// out[j][g], descending, zeros behind them.  A logit that at least k of the 256
// threads' own maxima reach bounds them from below, so that of a part's words little
// more than k are ranked against one another.  Where equal logits bring more words
// to it than the list holds, the bound is the k-th largest of the maxima as whole
// words: then at most k threads' all.  A workgroup's parts are of a size that gives
// the card one or two each; bound by the latency of its loads and six barriers: 4.4
// us for a row of 32000 in 32 parts, 8.7 for 25 rows of 152064 (1.7 TB/s).
template <int E>
__global__ __launch_bounds__(256) void k_part(Row a, u64 *__restrict__ out) {
    __shared__ __attribute__((aligned(16))) uint32_t best[256];
    __shared__ __attribute__((aligned(16))) u64 bestw[256];
    __shared__ __attribute__((aligned(16))) u64 list[4 * E * TK + 8];
    __shared__ u64 thr;
    __shared__ uint32_t cnt, low;
    const uint32_t tid = threadIdx.x, g = blockIdx.x, row = blockIdx.y, k = a.k;
    const float *const x = a.x + row * a.ld;
    const uint32_t first = g * a.part + 4 * tid, end = min(a.vocab, (g + 1) * a.part);
    float l[E][4];
#pragma unroll
    for (int e = 0; e < E; e++) load4(a, x, first + 1024 * e < end ? first + 1024 * e : a.vocab, l[e]);
    if (tid == 0) low = 0xFFFFFFFFu, cnt = 0, thr = 1;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; e++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) m = max(m, ord(l[e][j]));
    // each wavefront's ceil(k / 4)-th largest maximum, by bits (down to a step of
    // 2^-11 of it: a bound is enough); the least of the four is reached by k threads
    // at least
    uint32_t q = 0;
#pragma unroll
    for (int b = 31; b >= 12; b--) {
        const uint32_t c = q | 1u << b;
        if ((uint32_t)__popcll(__ballot(m >= c)) >= (k + 3) / 4) q = c;
    }
    best[tid] = m;
    __syncthreads();
    if ((tid & 63) == 0) atomicMin(&low, q);
    __syncthreads();
    if (low == 0) {
        // a wavefront with fewer words: the least of all maxima that fewer than k exceed
        uint32_t r = 0;
#pragma unroll 1
        for (uint32_t j = 0; j < 256; j += 32) {
            u32x4 v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = *reinterpret_cast<const u32x4 *>(best + j + 4 * e);
#pragma unroll
            for (int e = 0; e < 8; e++) r += (v[e][0] > m) + (v[e][1] > m) + (v[e][2] > m) + (v[e][3] > m);
        }
        __syncthreads();
        if (tid == 0) low = 0xFFFFFFFFu;
        __syncthreads();
        if (r < k) atomicMin(&low, m);
        __syncthreads();
    }
    const uint32_t lo = max(low, 1u);  // 0 where there are fewer than k words
    // the taken words to the list, one addition a wavefront for each of its words
    auto collect = [&](auto takes) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t i = first + 1024 * e;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const u64 w = word(l[e][j], i + j);
                const u64 who = __ballot(takes(w));
                if (!who) continue;
                uint32_t at = 0;
                if ((tid & 63) == 0) at = atomicAdd(&cnt, (uint32_t)__popcll(who));
                at = __builtin_amdgcn_readfirstlane(at) + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                if (takes(w) && at < 4 * E * TK) list[at] = w;
            }
        }
    };
    collect([&](u64 w) { return (uint32_t)(w >> 32) >= lo; });
    __syncthreads();
    if (cnt > 4 * E * TK) {
        u64 mw = 0;
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) mw = max(mw, word(l[e][j], first + 1024 * e + j));
        bestw[tid] = mw;
        __syncthreads();
        if (tid == 0) cnt = 0;
        if (mw && above(bestw, 256, mw) == k - 1) thr = mw;
        __syncthreads();
        const u64 t = thr;
        collect([&](u64 w) { return w >= t; });
        __syncthreads();
    }
    const uint32_t n = cnt;
    if (tid < 8) list[n + tid] = 0;
    __syncthreads();
    u64 *const o = out + (size_t)row * a.parts * k + g;
    for (uint32_t i = tid; i < n; i += 256) {
        const u64 w = list[i];
        const uint32_t rank = above(list, n, w);
        if (rank < k) o[(size_t)rank * a.parts] = w;
    }
    for (uint32_t i = n + tid; i < k; i += 256) o[(size_t)i * a.parts] = 0;
}

// The parts' words merged and the token picked.  The k-th largest of the first
// ceil(k / parts) words of every part bounds the row's k-th from below; where
// many words reach it (a few parts hold all the large ones), the k-th is found
// by bisection instead of ranking each against each.  One wavefront then picks,
// two words a lane: no barriers between the sums.  Latency bounds it: 5.7 us a row,
// 6.8 for 25 rows.
__global__ __launch_bounds__(512) void k_pick(Row a, const u64 *__restrict__ in) {
    struct Kept {
        u64 w;
        uint32_t at, pad;
    };
    __shared__ __attribute__((aligned(16))) u64 list[PICK_MAX + 8];
    __shared__ __attribute__((aligned(16))) u64 head[MAX_PARTS + TK + 8];
    __shared__ __attribute__((aligned(16))) u64 sel[TK];
    __shared__ __attribute__((aligned(16))) Kept kept[TK + 4];
    __shared__ u64 thr;
    __shared__ uint32_t cnt, nsel;
    const uint32_t tid = threadIdx.x, row = blockIdx.x, k = a.k, C = a.parts * k;
    const uint32_t H = a.parts * ((k + a.parts - 1) / a.parts);
    in += (size_t)row * C;
    u64 v[PICK_MAX / 512];
#pragma unroll
    for (uint32_t e = 0; e < PICK_MAX / 512; e++) v[e] = tid + 512 * e < C ? in[tid + 512 * e] : 0ull;
    if (tid < H + 8) head[tid] = tid < H ? v[0] : 0ull;
    if (tid < TK) sel[tid] = 0;
    if (tid == 0) thr = 1, cnt = 0, nsel = 0;
    __syncthreads();
    if (tid < H && v[0] && above(head, H, v[0]) == k - 1) thr = v[0];
    __syncthreads();
    u64 t = thr;
#pragma unroll
    for (uint32_t e = 0; e < PICK_MAX / 512; e++)
        if (512 * e < C && v[e] >= t) list[atomicAdd(&cnt, 1u)] = v[e];
    __syncthreads();
    uint32_t n = cnt;
    if (n > 1024) {
        // the largest value that at least k words reach, bit by bit
        t = 0;
        for (int b = 63; b >= 0; b--) {
            const u64 c = t | 1ull << b;
            uint32_t r = 0;
            for (uint32_t i = tid; i < n; i += 512) r += list[i] >= c;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) r += __shfl_xor(r, o, 64);
            __syncthreads();
            if (tid == 0) cnt = 0;
            __syncthreads();
            if ((tid & 63) == 0) atomicAdd(&cnt, r);
            __syncthreads();
            if (cnt >= k) t = c;
        }
        for (uint32_t i = tid; i < n; i += 512)
            if (list[i] >= t) head[atomicAdd(&nsel, 1u)] = list[i];
        __syncthreads();
        n = nsel;
        if (tid < n) list[tid] = head[tid];
        __syncthreads();
    }
    if (tid < 8) list[n + tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += 512) {
        const u64 w = list[i];
        const uint32_t r = above(list, n, w);
        if (r < k) sel[r] = w;
    }
    __syncthreads();
    if (tid >= 64) return;
    n = min(n, k);
    if (n == 0) {
        if (tid == 0) emit(a, row, 0xFFFFFFFFu, 0.f);
        return;
    }
    // lane i: words 2 i and 2 i + 1 of the order
    const float top = word_logit(sel[0]);
    u64 f[2], w[2];
    double p[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        w[e] = sel[2 * tid + e];
        p[e] = w[e] ? weight(word_logit(w[e]), top, a.inv_t) : 0.0;
        f[e] = fixed(p[e]);
    }
    const u64 inc = wave_scan(f[0] + f[1]);
    const double want = (double)a.top_p * (double)lane_value(inc, 63);
    u64 before = inc - f[0] - f[1], sum = 0, kf[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const bool keep = w[e] && ((tid == 0 && e == 0) || ((a.top_p >= 1.f || (double)before < want) && p[e] >= (double)a.min_p));
        before += f[e];
        kf[e] = keep ? f[e] : 0ull;
        sum += kf[e];
        kept[2 * tid + e] = Kept{kf[e], word_index(w[e]), 0};
    }
    if (tid < 4) kept[TK + tid] = Kept{0, 0, 0};
    sum = lane_value(wave_scan(sum), 63);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // a word's sum in index order, over the kept words
    u64 upto[2] = {0, 0};
    const uint32_t i0 = word_index(w[0]), i1 = word_index(w[1]);
    for (uint32_t j = 0; j < n; j += 4) {
        Kept q[4];
#pragma unroll
        for (int e = 0; e < 4; e++) q[e] = kept[j + e];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            upto[0] += q[e].at <= i0 ? q[e].w : 0ull;
            upto[1] += q[e].at <= i1 ? q[e].w : 0ull;
        }
    }
    const u64 past = target(a, row, sum);
    uint32_t c = 0xFFFFFFFFu;
    if (kf[0] && upto[0] > past) c = i0;
    if (kf[1] && upto[1] > past) c = min(c, i1);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c = min(c, (uint32_t)__shfl_xor(c, o, 64));
    if (kf[0] && i0 == c) emit(a, row, c, (float)(p[0] * ONE / (double)sum));
    if (kf[1] && i1 == c) emit(a, row, c, (float)(p[1] * ONE / (double)sum));
}

// ---- any top_k --------------------------------------------------------------
// What a row's workspace holds besides the parts' ranges and sums.
struct Hist {
    u64 mass[NB];
    uint32_t count[NB];
};
struct Cut {  // where the cuts fall (k_collect's first workgroup, for k_finish)
    // the bins of the list: top-p's cut is in b_lo..b_hi, top-k's in bk (NB: none);
    // words of bins before b_lo are kept
    uint32_t b_lo, b_hi, bk;
    uint32_t rank_k;  // words of bk that top-k keeps
    u64 before_lo, before_k;
};
struct Work {
    uint2 *range;      // [rows][parts] {largest, smallest} ord, 0: none
    u64 *sum;          // [rows][parts]
    Hist *hist;        // [rows]
    Cut *cut;          // [rows]
    u64 *list;         // [rows][LIST]
    uint32_t *n_list;  // [rows]
};

__device__ __forceinline__ bool cuts(const Row &a) { return a.k || a.top_p < 1.f; }

// The words of part g, four a thread at a time and the next four in flight;
// f(logit, index), where words below `least` may be left out
template <typename F>
__device__ __forceinline__ void for_words(const Row &a, uint32_t row, uint32_t g, float least, F f) {
    const float *const x = a.x + row * a.ld;
    const uint32_t end = min(a.vocab, (g + 1) * a.part);
    uint32_t i = g * a.part + 4 * threadIdx.x;
    float l[4], n[4];
    load4(a, x, i < end ? i : a.vocab, l);
#pragma unroll 1
    for (; i < end; i += 4 * WG) {
        load4(a, x, i + 4 * WG < end ? i + 4 * WG : a.vocab, n);
        if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= least)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) f(l[j], i + j);
#pragma unroll
        for (int j = 0; j < 4; j++) l[j] = n[j];
    }
}
// sum over the workgroup, in every thread
template <typename T>
__device__ __forceinline__ T wg_sum(T v, T (&sh)[WG / 64]) {
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = 0;
#pragma unroll
    for (uint32_t i = 0; i < WG / 64; i++) r += sh[i];
    return r;
}

// The largest and the least logit that can be taken, by part; it clears the
// histogram too.  3.6 us for a row of 152064, 12 for 64 rows of 248320 (5.3 TB/s: the
// read of the row is all it does).
__global__ __launch_bounds__(WG) void k_range(Row a, Work w) {
    __shared__ uint32_t mx, mn;
    const uint32_t tid = threadIdx.x, g = blockIdx.x, row = blockIdx.y;
    if (cuts(a)) {
        for (uint32_t i = g * WG + tid; i < NB; i += a.parts * WG) w.hist[row].mass[i] = 0, w.hist[row].count[i] = 0;
        if (g == 0 && tid == 0) w.n_list[row] = 0;
    }
    if (tid == 0) mx = 0, mn = 0xFFFFFFFFu;
    uint32_t hi = 0, lo = 0xFFFFFFFFu;
    for_words(a, row, g, -INFINITY, [&](float l, uint32_t) {
        const uint32_t k = ord(l);
        hi = max(hi, k);
        lo = min(lo, k - 1);  // 0, never taken, is the largest
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        hi = max(hi, (uint32_t)__shfl_xor(hi, o, 64));
        lo = min(lo, (uint32_t)__shfl_xor(lo, o, 64));
    }
    __syncthreads();
    if ((tid & 63) == 0) atomicMax(&mx, hi), atomicMin(&mn, lo);
    __syncthreads();
    if (tid == 0) w.range[(size_t)row * a.parts + g] = make_uint2(mx, mn + 1);
}

// the row's largest logit and the bins' scale, the same in every wavefront
struct Scale {
    float top, inv;
    bool any;
};
__device__ __forceinline__ Scale row_scale(const Row &a, const Work &w, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    uint2 r = make_uint2(0u, 0u);
    if (lane < a.parts) r = w.range[(size_t)row * a.parts + lane];
    r.y -= 1;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        r.x = max(r.x, (uint32_t)__shfl_xor(r.x, o, 64));
        r.y = min(r.y, (uint32_t)__shfl_xor(r.y, o, 64));
    }
    Scale s;
    s.any = r.x != 0;
    s.top = unord(r.x);
    // a word 30 T below the top weighs less than 2^-43: the bins end there
    const float width = fminf(s.top - unord(r.y + 1), 30.f * a.temp);
    s.inv = width > 0.f ? (float)(NB - 1) / width : 0.f;
    return s;
}
// monotone in l (each step rounds monotonically); NB: never taken
__device__ __forceinline__ uint32_t bin_of(float l, const Scale &s) {
    if (!(l > -INFINITY)) return NB;
    return l == s.top ? 0u : (uint32_t)fminf((s.top - l) * s.inv, (float)(NB - 1));
}

// Words (and with MASS their weights, where the list may not hold every word that
// counts) by bin: first in LDS, then added to the row's with whole-number atomics, whose
// order changes nothing.  5.4 us for a row of 152064 with weights, 14 for 64 rows of
// 248320 without.
template <bool MASS>
__global__ __launch_bounds__(WG) void k_hist(Row a, Work w) {
    __shared__ u64 mass[MASS ? NB : 1];
    __shared__ uint32_t count[NB];
    const uint32_t tid = threadIdx.x, g = blockIdx.x, row = blockIdx.y;
    const bool counts = a.k != 0;
    static_assert(NB == WG, "a thread clears and adds a bin");
    if constexpr (MASS) mass[tid] = 0;
    count[tid] = 0;
    const Scale s = row_scale(a, w, row);
    __syncthreads();
    for_words(a, row, g, -INFINITY, [&](float l, uint32_t) {
        const uint32_t b = bin_of(l, s);
        if (b == NB) return;
        if constexpr (MASS) {
            const u64 f = fixed(weight(l, s.top, a.inv_t));
            if (f) atomicAdd(&mass[b], f);
        }
        if (counts) atomicAdd(&count[b], 1u);
    });
    __syncthreads();
    Hist &h = w.hist[row];
    if constexpr (MASS)
        if (mass[tid]) atomicAdd(&h.mass[tid], mass[tid]);
    if (count[tid]) atomicAdd(&h.count[tid], count[tid]);
}

// the bins of the cuts from the row's histogram, a bin a thread
__device__ __forceinline__ Cut find_cuts(const Row &a, const Hist &h, u64 (&ms)[WG / 64], uint32_t (&cs)[WG / 64], u64 &after_k, Cut &sh) {
    const uint32_t tid = threadIdx.x;
    const u64 m = a.listed ? 0ull : h.mass[tid];
    const uint32_t c = h.count[tid];
    // sums of the bins before: within the wavefront, then over the wavefronts
    const u64 im = wave_scan(m);
    const uint32_t ic = wave_scan(c);
    if ((tid & 63) == 63) ms[tid >> 6] = im, cs[tid >> 6] = ic;
    __syncthreads();
    u64 total = 0, before = im - m;
    uint32_t n = 0, nb = ic - c;
#pragma unroll
    for (uint32_t i = 0; i < WG / 64; i++) {
        before += i < tid >> 6 ? ms[i] : 0ull;
        nb += i < tid >> 6 ? cs[i] : 0u;
        total += ms[i];
        n += cs[i];
    }
    // top-k's bin: the first that brings the count to k
    const bool cut_k = a.k && n > a.k;
    if (tid == 0) {
        sh.b_lo = sh.b_hi = NB;
        sh.before_lo = 0;
        if (!cut_k) sh.bk = NB, sh.rank_k = 0, sh.before_k = after_k = total;
    }
    if (cut_k && nb < a.k && nb + c >= a.k) {
        sh.bk = tid;
        sh.rank_k = a.k - nb;
        sh.before_k = before;
        after_k = before + m;
    }
    __syncthreads();
    if (a.listed) {
        if (tid == 0) sh.b_lo = 0, sh.b_hi = sh.bk, sh.before_k = 0;
    } else if (a.top_p < 1.f) {
        // K's sum is between its sums before and after top-k's bin: top-p's cut is in
        // the bins that bring the sum to top_p times either
        const double lo = (double)a.top_p * (double)sh.before_k, hi = (double)a.top_p * (double)after_k;
        const u64 nx = before + m;
        if (((double)before < lo || tid == 0) && (double)nx >= lo) sh.b_lo = tid, sh.before_lo = before;
        if (((double)before < hi || tid == 0) && (double)nx >= hi) sh.b_hi = tid;
    }
    __syncthreads();
    if (tid == 0 && !a.listed) {
        sh.b_lo = min(sh.b_lo, sh.bk);
        sh.b_hi = min(sh.b_hi, sh.bk);
        if (sh.b_lo == sh.bk) sh.before_lo = sh.before_k;  // top-k's bin alone where there is no top-p
    }
    __syncthreads();
    return sh;
}

__device__ __forceinline__ bool in_cuts(uint32_t b, const Cut &c) { return b < NB && ((b >= c.b_lo && b <= c.b_hi) || b == c.bk); }

// The words of the cuts' bins into the row's list, the sums of the words above them
// by part: what k_finish needs to find a cut without the row.  7.2 us for a row of
// 152064; 19 for 64 rows of 248320, listed.
__global__ __launch_bounds__(WG) void k_collect(Row a, Work w) {
    __shared__ u64 ms[WG / 64], put[LIST], after_k;
    __shared__ uint32_t cs[WG / 64], base, cnt, got;
    __shared__ Cut cut;
    const uint32_t tid = threadIdx.x, g = blockIdx.x, row = blockIdx.y;
    const Scale s = row_scale(a, w, row);
    Cut c = {NB, NB, NB, 0, 0, 0};
    if (tid == 0) cnt = got = 0;
    if (cuts(a)) {
        c = find_cuts(a, w.hist[row], ms, cs, after_k, cut);
        if (g == 0 && tid == 0) w.cut[row] = c;
    }
    __syncthreads();
    // Words below every bin that counts are passed over without their bin: a bin's
    // logits are not below this (the second term covers the roundings of bin_of, of
    // a bin's width, and of this difference)
    float least = -INFINITY;
    const uint32_t last = c.bk < NB ? c.bk : c.b_hi;
    if (last < NB - 1 && s.inv > 0.f && s.top < INFINITY) {
        const float d = (float)(last + 2) / s.inv;
        least = s.top - d - 0x1p-20f * (fabsf(s.top) + d);
    }
    // the words of bins that count are gathered and then weighed all at once (one by
    // one, every wavefront would wait for each of its few); too many go by in line
    const uint32_t after = min(last + 1, NB);
    u64 sum = 0;
    auto weigh = [&](float l) {
        const double v = weight(l, s.top, a.inv_t);
        if (v >= (double)a.min_p || l == s.top) sum += fixed(v);
    };
    for_words(a, row, g, least, [&](float l, uint32_t i) {
        if (bin_of(l, s) >= after) return;
        const uint32_t at = atomicAdd(&got, 1u);
        if (at < LIST) put[at] = word(l, i);
    });
    __syncthreads();
    const uint32_t n = got;
    __syncthreads();
    if (n <= LIST) {
        for (uint32_t i0 = 0; i0 < n; i0 += WG) {
            const uint32_t i = i0 + tid;
            const u64 v = i < n ? put[i] : 0ull;
            const float l = word_logit(v);
            const uint32_t b = i < n ? bin_of(l, s) : NB;
            if (b < c.b_lo) weigh(l);
            __syncthreads();  // put's first words make room for the list's
            if (b >= c.b_lo && in_cuts(b, c)) put[atomicAdd(&cnt, 1u)] = v;
            __syncthreads();
        }
    } else {
        for_words(a, row, g, least, [&](float l, uint32_t i) {
            const uint32_t b = bin_of(l, s);
            if (b < c.b_lo) {
                weigh(l);
            } else if (in_cuts(b, c)) {
                const uint32_t at = atomicAdd(&cnt, 1u);
                if (at < LIST) put[at] = word(l, i);
            }
        });
    }
    // the part's words behind those of other parts; a row with more than LIST
    // is counted in full and not read from the list
    __syncthreads();
    if (tid == 0 && cnt) base = atomicAdd(&w.n_list[row], cnt);
    __syncthreads();
    if (cnt)
        for (uint32_t i = tid; i < min(cnt, LIST) && base + i < LIST; i += WG) w.list[(size_t)row * LIST + base + i] = put[i];
    sum = wg_sum(sum, ms);
    if (tid == 0) w.sum[(size_t)row * a.parts + g] = sum;
}

// size (1024 or 2048) words sorted, largest first, by a workgroup
// of WG: a bitonic network.  A pair no more than 64 apart is in its wavefront's
// own 128 words, so that only the wider steps wait for the workgroup.
__device__ __forceinline__ void sort_words(u64 *list, uint32_t size) {
    const uint32_t t = threadIdx.x;
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            if (2 * t < size) {
                const uint32_t i = 2 * t - (t & (j - 1)), p = i + j;
                const u64 x = list[i], y = list[p];
                const bool down = (i & k) == 0 || k == size;
                if (x < y == down) list[i] = y, list[p] = x;
            }
            if (j > 64 || (j == 1 && k >= 128))
                __syncthreads();
            else
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
}

// n of list's words (up to LIST) sorted, largest first: a few are ranked against one
// another, many go through the network
__device__ __forceinline__ void order_words(u64 *list, uint32_t n) {
    const uint32_t tid = threadIdx.x;
    if (n <= 512) {
        if (tid < 8) list[n + tid] = 0;
        __syncthreads();
        const u64 v = tid < n ? list[tid] : 0ull;
        const uint32_t rank = tid < n ? above(list, n, v) : 0;
        __syncthreads();
        if (tid < n) list[rank] = v;
        __syncthreads();
    } else {
        const uint32_t size = n <= 1024 ? 1024 : 2048;
        for (uint32_t i = n + tid; i < size; i += WG) list[i] = 0;
        __syncthreads();
        sort_words(list, size);
    }
}

// The cuts among the collected words, the kept words' sums by part, and the
// token.  Only the words of the bins that the cuts fall in are ordered.  Where more
// of them than the list holds share those bins (equal logits by the thousand), the
// cuts are found bit by bit over the row itself.  One workgroup a row, whose barriers
// bound it: 9.4 us for a row of 152064, 11 for 64 rows of 248320 (31 with the whole
// list sorted).
__global__ __launch_bounds__(WG) void k_finish(Row a, Work w) {
    __shared__ __attribute__((aligned(16))) u64 list[LIST + 8];
    __shared__ u64 mass_of[NB];
    __shared__ uint32_t cnt, bin_p;
    __shared__ u64 before_p;
    __shared__ u64 part[64], red[WG / 64], thr;
    __shared__ uint32_t redc[WG / 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
    const float *const x = a.x + row * a.ld;
    const bool cut = cuts(a);
    // the list's first words are read before its length is known
    const u64 early = cut ? w.list[(size_t)row * LIST + tid] : 0ull;
    Cut c = {NB, NB, NB, 0, 0, 0};
    uint32_t n = 0;
    if (cut) {
        c = w.cut[row];
        n = w.n_list[row];
    }
    const Scale s = row_scale(a, w, row);
    if (!s.any) {
        if (tid == 0) emit(a, row, 0xFFFFFFFFu, 0.f);
        return;
    }
    if (tid < 64) part[tid] = tid < a.parts ? w.sum[(size_t)row * a.parts + tid] : 0ull;
    if (tid == 0) thr = ~0ull;
    auto mass = [&](u64 v) { return fixed(weight(word_logit(v), s.top, a.inv_t)); };
    if (cut && n <= LIST) {
        u64 v[2], f[2] = {0, 0}, thr_k = 0;
        double wd[2] = {0.0, 0.0};
        uint32_t b[2] = {NB, NB};
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t i = tid + WG * e;
            v[e] = i >= n ? 0ull : e == 0 ? early : w.list[(size_t)row * LIST + i];
            if (!v[e]) continue;
            b[e] = bin_of(word_logit(v[e]), s);
            wd[e] = weight(word_logit(v[e]), s.top, a.inv_t);
            f[e] = fixed(wd[e]);
        }
        // the words that `takes` says, in order
        auto gather = [&](auto takes) __attribute__((always_inline)) {
            __syncthreads();
            if (tid == 0) cnt = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (takes(e)) list[atomicAdd(&cnt, 1u)] = v[e];
            __syncthreads();
            const uint32_t m = cnt;
            order_words(list, m);
            return m;
        };
        if (c.bk < NB) {
            gather([&](int e) { return b[e] == c.bk; });
            thr_k = list[c.rank_k - 1];
        }
        auto in_k = [&](int e) { return v[e] && v[e] >= thr_k; };
        if (a.top_p < 1.f) {
            u64 m = 0;
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (in_k(e) && (a.listed || b[e] == c.bk)) m += f[e];
            const double want = (double)a.top_p * (double)(c.before_k + wg_sum(m, red));
            if (a.listed) {
                // the bin that the cut is in, from these words' weights by bin
                mass_of[tid] = 0;
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (in_k(e)) atomicAdd(&mass_of[b[e]], f[e]);
                __syncthreads();
                const u64 mine = mass_of[tid], up = wave_scan(mine);
                if (lane == 63) red[tid >> 6] = up;
                __syncthreads();
                u64 before = up - mine;
#pragma unroll
                for (uint32_t k = 0; k < WG / 64; k++) before += k < tid >> 6 ? red[k] : 0ull;
                if (((double)before < want || tid == 0) && (double)(before + mine) >= want) bin_p = tid, before_p = before;
                __syncthreads();
                c.b_lo = c.b_hi = bin_p;
                c.before_lo = before_p;
            }
            const uint32_t sub = gather([&](int e) { return in_k(e) && b[e] >= c.b_lo && b[e] <= c.b_hi; });
            // the words before which less than top-p's share has been, two a thread
            u64 x[2], g[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                x[e] = 2 * tid + e < sub ? list[2 * tid + e] : 0ull;
                g[e] = x[e] ? mass(x[e]) : 0ull;
            }
            const u64 up = wave_scan(g[0] + g[1]);
            if (lane == 63) red[tid >> 6] = up;
            __syncthreads();
            u64 before = c.before_lo + up - g[0] - g[1];
#pragma unroll
            for (uint32_t k = 0; k < WG / 64; k++) before += k < tid >> 6 ? red[k] : 0ull;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const bool keep = x[e] && (!before || (double)before < want);
                before += g[e];
                // they are the first ones: the least of a wavefront's is its last
                const u64 who = __ballot(keep);
                if (keep && lane == 63u - __clzll(who)) atomicMin(&thr, x[e]);
            }
        } else if (tid == 0) {
            thr = thr_k ? thr_k : 1;
        }
        __syncthreads();
        const u64 t = thr;
        if (a.listed) {
            // every kept word is here: their sums by index, NB stretches of the vocabulary,
            // the stretch that the token is in, and the token among its words
            mass_of[tid] = 0;
            __syncthreads();
            const uint32_t span = (a.vocab + NB - 1) / NB;
            u64 kf[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const bool kept = v[e] && (b[e] < c.b_lo || (b[e] <= c.b_hi && v[e] >= t)) && (wd[e] == 1.0 || wd[e] >= (double)a.min_p);
                kf[e] = kept ? f[e] : 0ull;
                if (kf[e]) atomicAdd(&mass_of[word_index(v[e]) / span], kf[e]);
            }
            __syncthreads();
            const u64 mine = mass_of[tid], up = wave_scan(mine);
            if (lane == 63) red[tid >> 6] = up;
            __syncthreads();
            u64 at = up - mine, sum = 0;
#pragma unroll
            for (uint32_t k = 0; k < WG / 64; k++) {
                at += k < tid >> 6 ? red[k] : 0ull;
                sum += red[k];
            }
            const u64 past = target(a, row, sum);
            if (at <= past && at + mine > past) bin_p = tid, before_p = at;
            __syncthreads();
            const uint32_t stretch = bin_p;
            const u64 before = before_p;
            const uint32_t m = gather([&](int e) { return kf[e] && word_index(v[e]) / span == stretch; });
            for (uint32_t i = tid; i < m; i += WG) {
                const uint32_t index = word_index(list[i]);
                u64 r = before;
                for (uint32_t j = 0; j < m; j++) r += word_index(list[j]) < index ? mass(list[j]) : 0ull;
                const double wi = weight(word_logit(list[i]), s.top, a.inv_t);
                if (r <= past && r + fixed(wi) > past) emit(a, row, index, (float)(wi * ONE / (double)sum));
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (v[e] && (b[e] < c.b_lo || (b[e] <= c.b_hi && v[e] >= t)) && (wd[e] == 1.0 || wd[e] >= (double)a.min_p))
                atomicAdd(&part[word_index(v[e]) / a.part], f[e]);
        __syncthreads();
    } else if (cut) {
        // bit by bit the largest value that enough of the bins' words reach
        auto count_at = [&](u64 v, uint32_t lo, uint32_t hi) {
            uint32_t r = 0;
            for (uint32_t i = tid; i < a.vocab; i += 1024) {
                const u64 q = word(x[i], i);
                const uint32_t b = bin_of(x[i], s);
                r += q >= v && b >= lo && b <= hi;
            }
            return wg_sum(r, redc);
        };
        auto mass_at = [&](u64 v, uint32_t lo, uint32_t hi) {
            u64 r = 0;
            for (uint32_t i = tid; i < a.vocab; i += 1024) {
                const u64 q = word(x[i], i);
                const uint32_t b = bin_of(x[i], s);
                if (q >= v && b >= lo && b <= hi) r += mass(q);
            }
            return wg_sum(r, red);
        };
        u64 tk = 0, sk = c.before_k;
        if (c.bk < NB)
            for (int b = 63; b >= 0; b--)
                if (count_at(tk | 1ull << b, c.bk, c.bk) >= c.rank_k) tk |= 1ull << b;
        if (c.bk < NB || a.listed) sk += mass_at(tk, a.listed ? 0 : c.bk, min(c.bk, NB - 1));
        u64 tp = tk;
        if (a.top_p < 1.f) {
            const double want = (double)a.top_p * (double)sk;
            tp = 0;
            for (int b = 63; b >= 0; b--) {
                const u64 r = c.before_lo + mass_at(max(tp | 1ull << b, tk), c.b_lo, c.b_hi);
                if (r && (double)r >= want) tp |= 1ull << b;
            }
            tp = max(tp, tk);
        }
        __syncthreads();
        if (tid == 0) thr = max(tp, 1ull);
        if (tid < 64) part[tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < a.vocab; i += 1024) {
            const uint32_t b = bin_of(x[i], s);
            if (b == NB || !(b < c.b_lo || (b <= c.b_hi && word(x[i], i) >= thr))) continue;
            const double v = weight(x[i], s.top, a.inv_t);
            const u64 f = fixed(v);
            if (f && (v >= (double)a.min_p || x[i] == s.top)) atomicAdd(&part[i / a.part], f);
        }
        __syncthreads();
    } else {
        __syncthreads();
    }
    // the part that the token is in: every wavefront adds up the parts, one a lane
    const u64 mine = part[lane], inc = wave_scan(mine);
    const u64 sum = lane_value(inc, 63), past = target(a, row, sum), t = thr;
    const uint32_t g = __ffsll((unsigned long long)__ballot(inc > past)) - 1;
    u64 run = lane_value(inc - mine, g);
    // ... and the token in it, 4096 words at a time
    const uint32_t end = min(a.vocab, (g + 1) * a.part);
    for (uint32_t i0 = g * a.part; i0 < end; i0 += 4096) {
        const uint32_t i = i0 + 4 * tid;
        float l[4];
        u64 f[4], m = 0;
        double v[4];
        load4(a, x, i < end ? i : a.vocab, l);
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t b = bin_of(l[j], s);
            f[j] = 0;
            if (b < NB && (b < c.b_lo || (b <= c.b_hi && word(l[j], i + j) >= t))) {
                v[j] = weight(l[j], s.top, a.inv_t);
                if (v[j] >= (double)a.min_p || l[j] == s.top) f[j] = fixed(v[j]);
            }
            m += f[j];
        }
        const u64 up = wave_scan(m);
        __syncthreads();
        if (lane == 63) red[tid >> 6] = up;
        __syncthreads();
        u64 at = run + up - m;
#pragma unroll
        for (uint32_t k = 0; k < 16; k++) {
            at += k < tid >> 6 ? red[k] : 0ull;
            run += red[k];
        }
        if (at <= past && at + m > past) {
            bool found = false;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                at += f[j];
                if (!found && at > past) {
                    found = true;
                    emit(a, row, i + j, (float)(v[j] * ONE / (double)sum));
                }
            }
        }
        if (run > past) break;
    }
}

// parts of a row for the first form: of one size, up to E pieces of 1024 words
uint32_t part_pieces(uint32_t vocab, uint32_t *e, uint32_t *part) {
    const uint32_t pieces = (vocab + 1023) / 1024;
    *e = pieces <= 64 ? 1 : pieces <= 128 ? 2 : pieces <= 256 ? 4 : 8;
    const uint32_t g = (pieces + *e - 1) / *e;
    *part = ((vocab + g - 1) / g + 3) / 4 * 4;
    return (vocab + *part - 1) / *part;
}
// ... and for the second: a workgroup per CU over all rows, four where k_finish
// goes over a part again (64 rows of 248320 words with top_k 1000 in 4, 8, 16 parts a
// row: k_collect 19, 24, 36 us); each at least 1024 words, a multiple of 4, so that
// rows stay aligned
uint32_t range_parts(uint32_t vocab, uint32_t rows, bool listed, uint32_t *part) {
    const uint32_t pieces = (vocab + 1023) / 1024;
    uint32_t g = ((listed ? 256 : 1024) + rows - 1) / rows;
    g = g < 4 ? 4 : g > 64 ? 64 : g;
    if (g > pieces) g = pieces;
    *part = ((vocab + g - 1) / g + 3) / 4 * 4;
    return (vocab + *part - 1) / *part;
}

// The first form as far as its lists go: at top_k 128 a row of 32000 takes 18 us
// against 23 with the second, 25 rows of 152064 26 against 36, 64 of 248320 46 against
// 51; at top_k 40 10 against 23 for the row of 32000.  Listed as far as half a list: the
// other half is for the rest of top-k's bin.
struct Plan {
    bool first, listed;
    uint32_t e, parts, part, k;
};
Plan plan(uint32_t rows, uint32_t vocab, const lrs_sampling &p) {
    Plan r = {};
    r.k = p.temperature == 0.f ? 1 : p.top_k >= vocab ? 0 : p.top_k;
    r.parts = part_pieces(vocab, &r.e, &r.part);
    r.first = r.k && r.k <= TK && r.parts <= MAX_PARTS && r.parts * r.k <= PICK_MAX;
    r.listed = !r.first && r.k && r.k <= LIST / 2;
    if (!r.first) r.parts = range_parts(vocab, rows, r.listed, &r.part);
    return r;
}

}  // namespace

size_t sample_work_bytes(uint32_t rows, uint32_t vocab, const lrs_sampling &p) {
    const Plan r = plan(rows, vocab, p);
    if (r.first) return (size_t)rows * r.parts * r.k * 8;
    return (size_t)rows * (r.parts * 16 + sizeof(Hist) + sizeof(Cut) + LIST * 8 + 8);
}

hipError_t launch_sample(const float *x, size_t ld, uint32_t rows, uint32_t vocab, const lrs_sampling &p, const float *u,
                         uint32_t *tok, float *prob, void *work, hipStream_t s, uint32_t *step, uint32_t *gen,
                         uint32_t gen_cap) {
    const Plan r = plan(rows, vocab, p);
    Row a = {};
    a.x = x;
    a.ld = ld;
    a.vocab = vocab;
    a.parts = r.parts;
    a.part = r.part;
    a.temp = p.temperature;
    a.inv_t = p.temperature > 0.f ? 1.0 / (double)p.temperature : 0.0;
    a.top_p = p.top_p;
    a.min_p = p.min_p;
    a.k = r.k;
    a.u = u;
    a.tok = tok;
    a.prob = prob;
    a.step = step;
    a.gen = gen;
    a.gen_cap = gen_cap;
    a.vec = (uintptr_t)x % 16 == 0 && ld % 4 == 0;
    if (r.first) {
        u64 *const w = (u64 *)work;
        const dim3 g(r.parts, rows);
        switch (r.e) {
        case 1: hipLaunchKernelGGL(k_part<1>, g, dim3(256), 0, s, a, w); break;
        case 2: hipLaunchKernelGGL(k_part<2>, g, dim3(256), 0, s, a, w); break;
        case 4: hipLaunchKernelGGL(k_part<4>, g, dim3(256), 0, s, a, w); break;
        default: hipLaunchKernelGGL(k_part<8>, g, dim3(256), 0, s, a, w); break;
        }
        hipLaunchKernelGGL(k_pick, dim3(rows), dim3(512), 0, s, a, (const u64 *)w);
        return hipGetLastError();
    }
    Work w;
    w.hist = (Hist *)work;
    w.cut = (Cut *)(w.hist + rows);
    w.list = (u64 *)(w.cut + rows);
    w.sum = w.list + (size_t)rows * LIST;
    w.range = (uint2 *)(w.sum + (size_t)rows * r.parts);
    w.n_list = (uint32_t *)(w.range + (size_t)rows * r.parts);
    const dim3 g(r.parts, rows);
    hipLaunchKernelGGL(k_range, g, dim3(WG), 0, s, a, w);
    a.listed = r.listed;
    if (a.listed)
        hipLaunchKernelGGL(k_hist<false>, g, dim3(WG), 0, s, a, w);
    else if (a.k || a.top_p < 1.f)
        hipLaunchKernelGGL(k_hist<true>, g, dim3(WG), 0, s, a, w);
    hipLaunchKernelGGL(k_collect, g, dim3(WG), 0, s, a, w);
    hipLaunchKernelGGL(k_finish, dim3(rows), dim3(WG), 0, s, a, w);
    return hipGetLastError();
}

}  // namespace lrs
