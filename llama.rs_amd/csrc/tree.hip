// tree.hip — a tree of drafted tokens in one pass: the rotation of q and k at
// given positions with the append to the f16 cache (k_rope_append), attention
// over the cache and over the drafted tokens that a bit mask lets each of them
// see (k_attn_tree, k_tree_merge), the walk down the tree along sampled tokens
// (k_tree_walk) and the move of the kept rows to consecutive slots
// (k_kv_keep).  No reference counterpart: its verify plan (resident_forward.rs:
// 3584-4170) takes a chain of tokens.
#include "gemm_pack.h"

#include <algorithm>

namespace lrs {

// ---- rotation + append ------------------------------------------------------
// Workgroup = a token's next 256 items of eight elements (or one pair, where
// rope_dim is no multiple of 8 or the rows are not 16-byte aligned); an item
// holds both elements of its pairs, so that q_out may be q.  The cos / sin of
// the token's pairs are made once per workgroup, in double up to the reduction
// to [-pi, pi]: the product of a far position and a frequency has more bits
// than a float.  q is read and written once, k and v read once and written in f16:
// a block of 512 tokens of the 32B shape (27 MB) takes 6.3 us, 4.3 TB/s, one token
// 2.8 (a launch).
template <bool VEC>
__global__ __launch_bounds__(256) void k_rope_append(RopeAppend a) {
    __shared__ float2 cs[128];
    const uint32_t tid = threadIdx.x, t = blockIdx.y, hd = a.head_dim, half = a.rope_dim / 2;
    constexpr uint32_t IT = VEC ? 8 : 2;
    const uint32_t per = hd / IT, item = blockIdx.x * 256 + tid;
    const uint32_t head = item / per, j = item % per, heads = a.n_head + 2 * a.n_kv;
    const bool act = head < heads;
    const int kind = head < a.n_head ? 0 : head < a.n_head + a.n_kv ? 1 : 2;
    const uint32_t hh = kind == 0 ? head : kind == 1 ? head - a.n_head : head - a.n_head - a.n_kv;
    const float *const src = kind == 0 ? a.q + t * a.ldq : kind == 1 ? a.k + t * a.ldk : a.v + t * a.ldv;
    const float *const bias = kind == 0 ? a.bq : kind == 1 ? a.bk : a.bv;
    // the item's two groups of IT / 2 elements: d0.., d1..
    const bool rot = kind < 2 && (a.halves ? j < half / (IT / 2) : true);
    uint32_t d0, d1;
    if (kind < 2 && a.halves) {
        d0 = rot ? j * (IT / 2) : a.rope_dim + (j - half / (IT / 2)) * IT;
        d1 = rot ? d0 + half : d0 + IT / 2;
    } else {
        d0 = j * IT;
        d1 = d0 + IT / 2;
    }
    float x[IT];
    if (act) {
        const float *const p = src + (size_t)hh * hd;
        if constexpr (VEC) {
            const float4 u = *reinterpret_cast<const float4 *>(p + d0), v = *reinterpret_cast<const float4 *>(p + d1);
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        } else {
            x[0] = p[d0], x[1] = p[d1];
        }
        if (bias)
#pragma unroll
            for (uint32_t e = 0; e < IT; e++) x[e] += bias[hh * hd + (e < IT / 2 ? d0 + e : d1 + e - IT / 2)];
    }
    if (tid < half) {
        const uint32_t pos = a.pos[t];
        const float f = a.freq[tid];
        float r;
        if (a.f32_angle) {
            r = (float)pos * f;
        } else {
            const double th = (double)pos * (double)f, n = rint(th * 0.15915494309189535);
            r = (float)fma(n, -2.4492935982947064e-16, fma(n, -6.283185307179586, th));
        }
        float sn, c;
        sincosf(r, &sn, &c);
        cs[tid] = make_float2(c * a.scale, sn * a.scale);
    }
    __syncthreads();
    if (!act) return;
    if (kind < 2) {
        if (a.halves) {
            if (rot) {
#pragma unroll
                for (uint32_t e = 0; e < IT / 2; e++) {
                    const float2 c = cs[d0 + e];
                    const float u = x[e], v = x[e + IT / 2];
                    x[e] = u * c.x - v * c.y;
                    x[e + IT / 2] = u * c.y + v * c.x;
                }
            }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < IT; e += 2) {
                if (d0 + e >= a.rope_dim) break;
                const float2 c = cs[(d0 + e) / 2];
                const float u = x[e], v = x[e + 1];
                x[e] = u * c.x - v * c.y;
                x[e + 1] = u * c.y + v * c.x;
            }
        }
    }
    if (kind == 0) {
        float *const o = a.q_out + ((size_t)t * a.n_head + hh) * hd;
        if constexpr (VEC) {
            *reinterpret_cast<float4 *>(o + d0) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(o + d1) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            o[d0] = x[0], o[d1] = x[1];
        }
        return;
    }
    const uint32_t slot = a.slot[t];
    if (slot >= a.rows) return;  // a padded token
    _Float16 *const o = (kind == 1 ? a.kc : a.vc) + ((size_t)hh * a.rows + slot) * hd;
    if constexpr (VEC) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<f16x4 *>(o + d0) = f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        *reinterpret_cast<f16x4 *>(o + d1) = f16x4{(_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]};
    } else {
        o[d0] = (_Float16)x[0], o[d1] = (_Float16)x[1];
    }
}

hipError_t launch_rope_append(const RopeAppend &a, hipStream_t s) {
    if (a.n == 0 || a.rope_dim > 256 || a.rope_dim > a.head_dim) return hipErrorInvalidValue;
    auto al = [](const void *p, size_t ld) { return (uintptr_t)p % 16 == 0 && ld % 4 == 0; };
    const bool vec = a.rope_dim % 8 == 0 && al(a.q, a.ldq) && al(a.k, a.ldk) && al(a.v, a.ldv) && al(a.q_out, 0) &&
                     (uintptr_t)a.kc % 8 == 0 && (uintptr_t)a.vc % 8 == 0;
    const uint32_t items = (a.n_head + 2 * a.n_kv) * (a.head_dim / (vec ? 8 : 2));
    hipLaunchKernelGGL(vec ? k_rope_append<true> : k_rope_append<false>, dim3((items + 255) / 256, a.n), dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---- attention --------------------------------------------------------------
// Rows: the n nodes' queries of the KV head's group, row = node * rep + head in
// the group, in tiles of 32.  A workgroup has T tiles and G groups of positions,
// a wavefront for each pair: group p takes every G-th chunk of 32 positions of the
// workgroup's share.  A chunk's K and V come to LDS with global_load_lds (the next
// chunk's are in flight during the current one's products), where the group's T
// wavefronts read them.  As in the prompt block's kernel S^T = K Q^T and
// O^T = V^T P^T run on v_mfma_f32_32x32x16_f16 with the exact f16 cache and q and p
// as f16 hi + lo (22 bits).  K's rows are XOR-swizzled (conflict-free 16-byte reads),
// V comes from its rows by transposing reads (ds_read_b64_tr_b16).
// The subtracted maximum follows the scores only when one exceeds it by 2^8: then
// the sums are rescaled; p stays below 2^8, which f32 sums and f16 pairs hold.
// Measured, attention + merge, 40 heads on 8 KV heads of 128: 64 nodes behind 130000
// positions 355 us (341 Gflop as two products: 0.96 PFLOP/s); 26 behind 3900 21 us and 8
// behind 333 11 us, of which a workgroup's fixed part (q, the first chunk from HBM,
// the sums through LDS) is 7 us, a chunk 1 us and the merge 4.  41 nodes, 24 heads on
// 4 KV heads of 256, behind 2047: 33 us, the fixed part 11 of them; q and O fill
// the registers there, and four wavefronts a workgroup (30 us for the kernel), two
// workgroups a CU (32) and one copy of the code for all chunks (32) gain nothing on
// two wavefronts (29).
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
typedef __fp16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __fp16 h16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) h16x4_t lds_h16x4_t;
typedef __attribute__((address_space(3))) void lds_void_t;

// the 32 positions from 32 c on that row `node` sees
__device__ __forceinline__ uint32_t seen_bits(const AttnTree &a, uint32_t node, uint32_t c) {
    const uint32_t W = (a.n + 31) / 32;
    auto word = [&](uint32_t j) -> uint32_t {
        if (j >= W) return 0u;
        const uint32_t left = a.n - 32 * j;
        const uint32_t have = left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1;
        if (a.mask) return a.mask[(size_t)node * W + j] & have;
        const uint32_t up = node + 1 > 32 * j ? node + 1 - 32 * j : 0;  // a chain: nodes 0..node
        return up >= 32 ? 0xFFFFFFFFu : (1u << up) - 1;
    };
    const uint32_t p0 = 32 * c;
    if (p0 >= a.len) {
        const uint32_t d = p0 - a.len, b = d & 31;
        return b ? (word(d >> 5) >> b) | word((d >> 5) + 1) << (32 - b) : word(d >> 5);
    }
    const uint32_t k = a.len - p0;
    return k >= 32 ? 0xFFFFFFFFu : ((1u << k) - 1) | word(0) << k;
}

// the larger of the two half wavefronts' x, in both
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// wavefronts per SIMD that the LDS of as many workgroups as fit allows, at most 2
// (the registers' limit at head_dim 128; 1 at 256)
constexpr int tree_waves(int HD, int T, int G) {
    const int lds = G * HD * 256 + G * T * 256;
    return HD < 256 && 163840 / lds * T * G >= 8 ? 2 : 1;
}

template <int HD, int T, int G>
__global__ __launch_bounds__(64 * T * G, tree_waves(HD, T, G)) void k_attn_tree(AttnTree a) {
    constexpr int KS = HD / 16;     // K-steps of S^T
    constexpr int OT = HD / 32;     // tiles of O^T = dims of a lane's V
    constexpr int NPR = HD / 8;     // 16-byte pieces of a row
    constexpr int NI = HD / 16;     // 1 KB loads of a chunk's K or V
    // A transposing read of 32 lanes takes 64 bytes of each of four rows: V's 16-byte
    // pieces are turned by the row (row >> VT & VM, times 4) so that those are in
    // different banks
    constexpr uint32_t VT = HD == 64 ? 1 : 0, VM = HD == 64 ? 1 : 3;
    // tiles of a check for values that are not finite: at head_dim 256 one, whose
    // registers are all taken (36 us with eight, 33 with one: 41 nodes behind 2047
    // positions, 24 heads on 4 KV heads), else all (26 nodes of the 32B shape behind
    // 3900 positions: no difference, but no spill)
    constexpr int OC = HD == 256 ? 1 : OT;
    // K, then V of a group's chunk of even and of odd rounds; the groups' sums at the end
    __shared__ __attribute__((aligned(16))) _Float16 buf0[G][64 * HD], buf1[G][64 * HD];
    __shared__ float2 wml[G][T * 32];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hf = lane >> 5, col = lane & 31;
    const uint32_t tw = wave % T, grp = wave / T;
    const uint32_t rep = a.n_head / a.n_kv, rows = a.n * rep, tgs = (a.tiles + T - 1) / T;
    // the KV head goes fastest, so that with eight of them an XCD keeps one
    // head's rows in its L2, then the tiles, which share them
    const uint32_t g = blockIdx.x % a.n_kv, tile = blockIdx.x / a.n_kv % tgs * T + tw, sp = blockIdx.x / a.n_kv / tgs;
    const uint32_t r0 = 32 * tile + col, r = min(r0, rows - 1);  // lanes past the rows compute a copy
    const uint32_t node = r / rep, h = g * rep + r % rep;
    const uint32_t P = a.len + a.n, nch = (P - 1) / 32 + 1;
    const uint32_t share = (nch + a.S - 1) / a.S, c0 = sp * share, c1 = min(c0 + share, nch);
    const _Float16 *const kb = a.kc + (size_t)g * a.rows * HD;
    const _Float16 *const vb = a.vc + (size_t)g * a.rows * HD;

    uint32_t v_at[OT];
    {
        const uint32_t row = 4 * hf + (lane >> 2 & 3);
#pragma unroll
        for (int t = 0; t < OT; t++)
            v_at[t] = row * HD + 8 * (4 * t ^ ((row >> VT & VM) << 2)) + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
    }
    // chunk c -> the even or odd rounds' buffer: slot s (16 B) of K holds row s / NPR, piece
    // (s % NPR) ^ (row % NPR).  Past the end: a row that is there.
    auto stage = [&](uint32_t c, const bool odd) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < (NI + T - 1) / T; i++) {
            const uint32_t j = i * T + tw;
            if (NI % T && j >= NI) break;
            const uint32_t sl = 64 * j + lane, row = sl / NPR, pc = sl % NPR;
            const size_t at = (size_t)min(32 * c + row, P - 1) * HD;
            __builtin_amdgcn_global_load_lds(kb + at + 8 * (pc ^ (row % NPR)), (lds_void_t *)((odd ? buf1[grp] : buf0[grp]) + 512 * j), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(vb + at + 8 * (pc ^ ((row >> VT & VM) << 2)), (lds_void_t *)((odd ? buf1[grp] : buf0[grp]) + 32 * HD + 512 * j), 16, 0, 0);
        }
    };
    // the same rounds for every group; the first `plain` of them are of positions
    // that every row sees.  The two buffers are objects of their own and the
    // plain rounds' parity is fixed, so that the compiler need not wait for the
    // loads into one before it reads the other
    const uint32_t first = c0 + grp;
    const uint32_t rounds = c1 > c0 ? (c1 - c0 + G - 1) / G : 0, whole = min(c1, a.len / 32);
    const uint32_t plain = whole > c0 ? (whole - c0) / G : 0;
    // what the row sees of its masked chunk: read a round ahead
    uint32_t seen = seen_bits(a, node, first + (plain & ~1u) * G);
    f16x8_t qh[KS], ql[KS];
    float qsc;
    {
        const float *const qp = a.q + ((size_t)node * a.n_head + h) * HD + 8 * hf;
        float qv[KS][8], qm = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const float4 u = *reinterpret_cast<const float4 *>(qp + 16 * k);
            const float4 v = *reinterpret_cast<const float4 *>(qp + 16 * k + 4);
            qv[k][0] = u.x, qv[k][1] = u.y, qv[k][2] = u.z, qv[k][3] = u.w;
            qv[k][4] = v.x, qv[k][5] = v.y, qv[k][6] = v.z, qv[k][7] = v.w;
        }
        // q's loads before the first chunk's: loads return in order
        if (first < c1) stage(first, false);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) qm = fmaxf(qm, fabsf(qv[k][e]));
        qm = half_max(qm);
        int ex;
        (void)frexpf(qm, &ex);
        ex = ex < -60 ? -60 : ex;
        // the scores' factor is positive (the maximum is taken before it): the
        // scale's sign goes into q
        const float sgn = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
        qsc = a.scale == 0.f ? 1.f : ldexpf(fabsf(a.scale) * 1.4426950408889634f, ex);  // in powers of two
        const float down = ldexpf(sgn, -ex);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = qv[k][e] * down;
                const _Float16 xh = (_Float16)x;
                qh[k][e] = xh;
                ql[k][e] = (_Float16)(x - (float)xh);
            }
    }
    f32x16_t o[OT];
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = 0.f;
    float m = -INFINITY, l = 0.f;  // l: of the lane's own positions
    // the products of the chunk in buffer b; masked (a constant): it has positions that some
    // rows do not see, the row's are `seen`
    auto chunk = [&](const bool masked, uint32_t seen, const _Float16 *b) __attribute__((always_inline)) {
        const _Float16 *const Kc = b, *const Vc = b + 32 * HD;
        const uint32_t mine = seen >> (4 * hf);
        f32x16_t sc;
#pragma unroll
        for (int i = 0; i < 16; i++) sc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const f16x8_t kf = *reinterpret_cast<const f16x8_t *>(Kc + 8 * (col * NPR + ((2 * k + hf) ^ (col % NPR))));
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[k], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[k], sc, 0, 0, 0);
        }
        // the lane's scores are positions 8 (i / 4) + 4 hf + i % 4
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; i++) sc[i] = mine >> (8 * (i >> 2) + (i & 3)) & 1 ? sc[i] : -INFINITY;
        }
        float cmax = sc[0];
#pragma unroll
        for (int i = 1; i < 16; i++) cmax = fmaxf(cmax, sc[i]);
        cmax = half_max(cmax) * qsc;
        if (__any(cmax > m + 8.f)) {
            const float mn = fmaxf(m, cmax);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < OT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[t][i] *= alpha;
        }
        // a row that has seen nothing yet has only -inf: any finite maximum gives zeros
        const float ms = m == -INFINITY ? 0.f : m;
        f16x8_t ph[2], pl[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], qsc, -ms));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i + 1], qsc, -ms));
            l += p0;
            l += p1;
            const f16x2_t hi = __builtin_amdgcn_cvt_pkrtz(p0, p1);
            const f16x2_t lo = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)hi[0], -1.f, p0), __builtin_fmaf((float)hi[1], -1.f, p1));
            ph[i >> 3][i & 7] = (_Float16)hi[0], ph[i >> 3][(i & 7) + 1] = (_Float16)hi[1];
            pl[i >> 3][i & 7] = (_Float16)lo[0], pl[i >> 3][(i & 7) + 1] = (_Float16)lo[1];
        }
        // the transposing read gives lane i of sixteen column i of four rows, from
        // addresses of four elements each: V of positions 16 s + 8 (j / 4) + 4 hf
        // + j % 4, slots j of step s, for dim 32 t + lane % 32
#pragma unroll
        for (int s = 0; s < 2; s++) {
            f16x8_t va[OT];
#pragma unroll
            for (int t = 0; t < OT; t++) {
                const _Float16 *const p = Vc + v_at[t] + 16 * s * HD;
                const h16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_h16x4_t *)p);
                const h16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_h16x4_t *)(p + 8 * HD));
#pragma unroll
                for (int j = 0; j < 4; j++) va[t][j] = (_Float16)lo[j], va[t][j + 4] = (_Float16)hi[j];
            }
            // a V that is not finite reaches the rows that see it alone: it is taken
            // out of the product (0 inf is NaN) and added where it is seen
            if (masked) {
#pragma unroll
                for (int t0 = 0; t0 < OT; t0 += OC) {
                    u16x2_t top = {0, 0};
#pragma unroll
                    for (int t = t0; t < t0 + OC; t++) {
                        const u16x8_t bits = __builtin_bit_cast(u16x8_t, va[t]) & (uint16_t)0x7FFF;
#pragma unroll
                        for (int j = 0; j < 8; j += 2) top = __builtin_elementwise_max(top, u16x2_t{bits[j], bits[j + 1]});
                    }
                    if (!__any(max(top[0], top[1]) >= 0x7C00)) continue;
                    f16x8_t one;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        one[j] = mine >> (16 * s + 8 * (j >> 2) + (j & 3)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
                    for (int t = t0; t < t0 + OC; t++) {
#pragma unroll 1
                        for (int kind = 0; kind < 3; kind++) {  // NaN, inf, -inf
                            f16x8_t is;
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                const _Float16 v = va[t][j];
                                const bool hit = kind == 0 ? v != v : v == (kind == 1 ? (_Float16)INFINITY : -(_Float16)INFINITY);
                                is[j] = hit ? (_Float16)1.0f : (_Float16)0.0f;
                            }
                            f32x16_t n;
#pragma unroll
                            for (int i = 0; i < 16; i++) n[i] = 0.f;
                            n = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, one, n, 0, 0, 0);
                            const float val = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (n[i] > 0.f) o[t][i] += val;
                        }
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            if (!(__builtin_fabsf16(va[t][j]) <= (_Float16)65504.0f)) va[t][j] = (_Float16)0.0f;
                    }
                }
            }
            // neighbouring products go to different sums
#pragma unroll
            for (int t = 0; t < OT; t++) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[t], pl[s], o[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < OT; t++) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[t], ph[s], o[t], 0, 0, 0);
        }
    };
    auto next = [&](uint32_t it, const bool odd) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (first + (it + 1) * G < c1) stage(first + (it + 1) * G, !odd);
    };
    uint32_t it = 0;
    for (; it + 1 < plain; it += 2) {
        next(it, false);
        chunk(false, 0xFFFFFFFFu, buf0[grp]);
        next(it + 1, true);
        chunk(false, 0xFFFFFFFFu, buf1[grp]);
    }
    for (; it < rounds; it++) {
        const uint32_t c = first + it * G, now = seen;
        next(it, it & 1);
        seen = seen_bits(a, node, c + G);
        if (c < c1) chunk(true, now, it & 1 ? buf1[grp] : buf0[grp]);
    }
    l += __shfl_xor(l, 32, 64);
    float M = m, L = l, f = 1.f;
    if constexpr (G > 1) {
        // the groups' sums over the common maximum
        if (hf == 0) wml[grp][tw * 32 + col] = make_float2(m, l);
        __syncthreads();  // and every group has read its last chunk
        M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < G; w++) M = fmaxf(M, wml[w][tw * 32 + col].x);
#pragma unroll
        for (int w = 0; w < G; w++) {
            const float2 p = wml[w][tw * 32 + col];
            if (p.y != 0.f) L += p.y * __builtin_amdgcn_exp2f(p.x - M);
        }
        f = l != 0.f ? __builtin_amdgcn_exp2f(m - M) : 0.f;
    }
    const size_t row_at = ((size_t)node * a.n_head + h) * HD;
    if (grp == 0 && hf == 0 && a.S > 1 && r0 < rows) a.ml[((size_t)sp * a.n + node) * a.n_head + h] = make_float2(M, L);
    f *= a.S > 1 ? 1.f : L != 0.f ? 1.f / L : 0.f;
    float *const out = a.S > 1 ? a.part + (size_t)sp * a.n * a.n_head * HD : a.out;
    // a lane's runs of four elements: at 32 t + 8 i + 4 hf
    auto run = [&](int t, int i) {
        return l != 0.f ? make_float4(o[t][4 * i] * f, o[t][4 * i + 1] * f, o[t][4 * i + 2] * f, o[t][4 * i + 3] * f)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    if constexpr (G == 1) {
        if (r0 >= rows) return;
#pragma unroll
        for (int t = 0; t < OT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<float4 *>(out + row_at + 32 * t + 8 * i + 4 * hf) = run(t, i);
        return;
    }
    // each group's tile t into its own buffer t (of 32 rows; the row's pieces of four
    // elements turned by the row, so that the lanes of a write are in different banks)
    static_assert(G == 1 || T <= 2, "a group has two buffers");
    float *const mine = reinterpret_cast<float *>(tw ? buf1[grp] : buf0[grp]) + col * HD;
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<float4 *>(mine + 4 * ((8 * t + 2 * i + hf) ^ (col % (HD / 4)))) = run(t, i);
    __syncthreads();
    for (uint32_t i = tid; i < T * 32 * (HD / 4); i += 64 * T * G) {
        const uint32_t q = i / (HD / 4), d = i % (HD / 4), row = 32 * (tile - tw) + q;
        if (row >= rows) break;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < G; w++) {
            const float4 x = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(q < 32 ? buf0[w] : buf1[w]) +
                                                               (q % 32) * HD + 4 * (d ^ (q % 32 % (HD / 4))));
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        *reinterpret_cast<float4 *>(out + ((size_t)(row / rep) * a.n_head + g * rep + row % rep) * HD + 4 * d) = v;
    }
}

// The workgroups' shares of a row joined: F threads (a power of two) for each 4
// elements, which take every F-th share.  Load latency bounds it: a thread's shares
// go by in fours.  3.9 us for 26 nodes of 40 heads of 128 in 10 shares, 6.6 for 64
// nodes.
__global__ __launch_bounds__(256) void k_tree_merge(AttnTree a, uint32_t hd, uint32_t F) {
    __shared__ float4 sv[256];
    __shared__ float2 sm[256];
    const uint32_t tid = threadIdx.x, e4 = hd / 4, per = e4 * F;
    const uint32_t f = tid % per / e4, e = 4 * (tid % e4);
    const size_t R = (size_t)a.n * a.n_head, r = (size_t)blockIdx.x * (256 / per) + tid / per, N = R * hd;
    float M = -INFINITY, L = 0.f, v[4] = {};
    if (r < R)
        for (uint32_t s0 = f; s0 < a.S; s0 += 4 * F) {
            float2 p[4];
            float4 x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t s = min(s0 + i * F, a.S - 1);
                p[i] = a.ml[s * R + r];
                x[i] = *reinterpret_cast<const float4 *>(a.part + s * N + r * hd + e);
                if (s0 + i * F >= a.S) p[i] = make_float2(-INFINITY, 0.f);
            }
            const float mn = fmaxf(M, fmaxf(fmaxf(p[0].x, p[1].x), fmaxf(p[2].x, p[3].x)));
            const float al = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
            L *= al;
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] *= al;
            M = mn;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (p[i].y == 0.f) continue;  // saw nothing
                const float w = __builtin_amdgcn_exp2f(p[i].x - M);
                L = fmaf(p[i].y, w, L);
                v[0] = fmaf(w, x[i].x, v[0]), v[1] = fmaf(w, x[i].y, v[1]);
                v[2] = fmaf(w, x[i].z, v[2]), v[3] = fmaf(w, x[i].w, v[3]);
            }
        }
    if (F > 1) {
        sv[tid] = make_float4(v[0], v[1], v[2], v[3]);
        sm[tid] = make_float2(M, L);
        __syncthreads();
        if (f) return;
        float mn = M;
        for (uint32_t i = 1; i < F; i++) mn = fmaxf(mn, sm[tid + i * e4].x);
        const float al = L != 0.f ? __builtin_amdgcn_exp2f(M - mn) : 0.f;
        L *= al;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = L != 0.f ? v[k] * al : 0.f;
        for (uint32_t i = 1; i < F; i++) {
            const float2 p = sm[tid + i * e4];
            const float4 x = sv[tid + i * e4];
            if (p.y == 0.f) continue;
            const float w = __builtin_amdgcn_exp2f(p.x - mn);
            L = fmaf(p.y, w, L);
            v[0] = fmaf(w, x.x, v[0]), v[1] = fmaf(w, x.y, v[1]), v[2] = fmaf(w, x.z, v[2]), v[3] = fmaf(w, x.w, v[3]);
        }
    }
    if (r >= R) return;
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    *reinterpret_cast<float4 *>(a.out + r * hd + e) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}

// Tiles and position groups of a workgroup, and shares of the positions: four
// wavefronts a workgroup (two at head_dim 256, whose buffers are twice as large),
// of two tiles where there are two; a workgroup per CU, and two (the second
// wavefront of a SIMD, whose products overlap the first's softmax) where a
// wavefront then still has eight chunks: 64 nodes of the 32B shape behind 130000
// positions 413 -> 369 us, 26 behind 3900 22 -> 26 us.  One tile and twice the groups
// where there are more tiles: 64 nodes 354 -> 578 us, 26 (five tiles) 22 -> 21, 8
// behind 333 10.8 -> 11.6, 41 at head_dim 256 33 -> 34.
struct TreeShape {
    uint32_t T, G, S;
};
static TreeShape tree_shape(uint32_t n, uint32_t len, uint32_t n_head, uint32_t n_kv, uint32_t hd) {
    const uint32_t tiles = (n * (n_head / n_kv) + 31) / 32, chunks = (len + n - 1) / 32 + 1;
    TreeShape r;
    r.T = tiles == 1 ? 1 : 2;
    r.G = hd == 256 ? 2 / r.T : 4 / r.T;
    const uint32_t wgs = (tiles + r.T - 1) / r.T * n_kv;
    const uint32_t full = hd < 256 && (uint64_t)chunks * wgs >= 512u * 8 * r.G ? 512 : 256;
    const uint32_t S = std::max(1u, std::min(full / wgs, (chunks + r.G - 1) / r.G));
    // no empty share
    const uint32_t share = (chunks + S - 1) / S;
    r.S = (chunks + share - 1) / share;
    return r;
}

size_t attn_tree_work_bytes(uint32_t n, uint32_t len, uint32_t n_head, uint32_t n_kv, uint32_t hd) {
    const uint32_t S = tree_shape(n, len, n_head, n_kv, hd).S;
    return S > 1 ? (size_t)S * n * n_head * (hd * 4 + 8) : 0;
}

hipError_t launch_attn_tree(AttnTree a, uint32_t hd, void *work, hipStream_t s) {
    if (a.n == 0 || a.n_kv == 0 || a.n_head == 0 || a.n_head % a.n_kv) return hipErrorInvalidValue;
    const TreeShape sh = tree_shape(a.n, a.len, a.n_head, a.n_kv, hd);
    a.tiles = (a.n * (a.n_head / a.n_kv) + 31) / 32;
    a.S = sh.S;
    if (a.S > 1) {
        if (!work) return hipErrorInvalidValue;
        a.part = (float *)work;
        a.ml = (float2 *)(a.part + (size_t)a.S * a.n * a.n_head * hd);
    }
    void (*fn)(AttnTree) = nullptr;
#define LRS_TREE(H, T_, G_) \
    if (hd == H && sh.T == T_ && sh.G == G_) fn = k_attn_tree<H, T_, G_>;
    LRS_TREE(64, 1, 4) LRS_TREE(64, 2, 2)
    LRS_TREE(128, 1, 4) LRS_TREE(128, 2, 2)
    LRS_TREE(256, 1, 2) LRS_TREE(256, 2, 1)
#undef LRS_TREE
    if (!fn) return hipErrorInvalidValue;
    hipLaunchKernelGGL(fn, dim3((a.tiles + sh.T - 1) / sh.T * a.n_kv * a.S), dim3(64 * sh.T * sh.G), 0, s, a);
    if (a.S > 1) {
        uint32_t F = 1;
        while (F < 1024 / hd && 4 * F < a.S) F *= 2;
        const uint32_t rows = 256 / (hd / 4 * F);
        hipLaunchKernelGGL(k_tree_merge, dim3((a.n * a.n_head + rows - 1) / rows), dim3(256), 0, s, a, hd, F);
    }
    return hipGetLastError();
}

// ---- the walk and the kept rows ---------------------------------------------
// From node 0 down: a node's sampled token is the next token; the walk goes on
// at the first child that drafted it.  out: {length of the walk, its tokens};
// path: its nodes.  One wavefront; a node's parent comes before it, so that
// the walk takes at most n steps.  A chain of dependent loads: 5.4 us for seven
// steps down a tree of 26.
__global__ __launch_bounds__(64) void k_tree_walk(const uint32_t *__restrict__ tokens, const uint32_t *__restrict__ parents,
                                                  const uint32_t *__restrict__ sampled, uint32_t n, uint32_t *__restrict__ out,
                                                  uint32_t *__restrict__ path) {
    const uint32_t lane = threadIdx.x;
    uint32_t cur = 0, k = 0;
    for (uint32_t step = 0; step < n; step++) {
        const uint32_t t = sampled[cur];
        if (lane == 0) {
            path[k] = cur;
            out[1 + k] = t;
        }
        k++;
        uint32_t next = n;
        for (uint32_t i = cur + 1 + lane; i < n; i += 64)
            if (parents[i] == cur && tokens[i] == t) {
                next = i;
                break;
            }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) next = min(next, (uint32_t)__shfl_xor(next, o, 64));
        if (next >= n) break;
        cur = next;
    }
    if (lane == 0) out[0] = k;
}

// Rows pos0 + path[i] of every layer's K and V to pos0 + i, i < *count.  A
// thread moves one 16-byte piece of every kept row of a head, eight rows in
// flight: path ascends and path[i] >= i, so no later read is of a row that an
// earlier write has replaced.  Latency: 3.7 us for seven rows of two layers.
__global__ __launch_bounds__(256) void k_kv_keep(_Float16 *kv, uint32_t planes, uint32_t hd, uint32_t ctx, uint32_t pos0,
                                                 const uint32_t *__restrict__ count, const uint32_t *__restrict__ path) {
    const uint32_t per = hd / 8, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= planes * per) return;
    _Float16 *const p = kv + ((size_t)(i / per) * ctx + pos0) * hd + 8 * (i % per);
    const uint32_t n = *count;
    for (uint32_t k = 0; k < n; k += 8) {
        uint4 v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            v[j] = *reinterpret_cast<const uint4 *>(p + (size_t)path[min(k + j, n - 1)] * hd);
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (k + j < n) *reinterpret_cast<uint4 *>(p + (size_t)(k + j) * hd) = v[j];
    }
}

hipError_t launch_tree_walk(const uint32_t *tokens, const uint32_t *parents, const uint32_t *sampled, uint32_t n,
                            uint32_t *out, uint32_t *path, hipStream_t s) {
    hipLaunchKernelGGL(k_tree_walk, dim3(1), dim3(64), 0, s, tokens, parents, sampled, n, out, path);
    return hipGetLastError();
}

hipError_t launch_kv_keep(_Float16 *kv, uint32_t planes, uint32_t hd, uint32_t ctx, uint32_t pos0, const uint32_t *count,
                          const uint32_t *path, hipStream_t s) {
    const uint32_t items = planes * (hd / 8);
    hipLaunchKernelGGL(k_kv_keep, dim3((items + 255) / 256), dim3(256), 0, s, kv, planes, hd, ctx, pos0, count, path);
    return hipGetLastError();
}

}  // namespace lrs
