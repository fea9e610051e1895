// tree.hip — a tree of drafted tokens in one pass: the rotation of q and k at
// given positions with the append to the f16 cache (k_rope_append), attention
// over the cache and over the drafted tokens that a bit mask lets each of them
// see (k_attn_tree, k_tree_merge), the walk down the tree along sampled tokens
// (k_tree_walk) and the move of the kept rows to consecutive slots
// (k_kv_keep).  No reference counterpart: its verify plan (resident_forward.rs:
// 3584-4170) takes a chain of tokens.
#include "gemm_pack.h"

namespace lrs {

// ---- rotation + append ------------------------------------------------------
// Workgroup = a token's next 256 items of eight elements (or one pair, where
// rope_dim is no multiple of 8 or the rows are not 16-byte aligned); an item
// holds both elements of its pairs, so that q_out may be q.  The cos / sin of
// the token's pairs are made once per workgroup, in double up to the reduction
// to [-pi, pi]: the product of a far position and a frequency has more bits
// than a float.
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
// the group, in tiles of 32.  A wavefront takes one tile and every NW-th chunk
// of 32 positions of its workgroup's share; the workgroup's wavefronts are
// merged through LDS, workgroups by k_tree_merge.  As in the prompt block's
// kernel S^T = K Q^T and O^T = V^T P^T run on v_mfma_f32_32x32x16_f16 with the
// exact f16 cache and q and p as f16 hi + lo (22 bits); here K and V come
// straight from the cache into the operand registers, with no LDS and no
// barrier in the loop: a lane holds 16 bytes of one position's K per K-step, and
// HD / 32 neighbouring dims of each of its positions' V, which it repacks
// two positions at a time; O^T tile t then holds dims HD / 32 * i + t.
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

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

template <int HD, int NW>
__global__ __launch_bounds__(64 * NW) void k_attn_tree(AttnTree a) {
    constexpr int KS = HD / 16;  // K-steps of S^T
    constexpr int OT = HD / 32;  // tiles of O^T = dims of a lane's V
    constexpr int LD = HD + 4;
    __shared__ __attribute__((aligned(16))) float osum[32 * LD];
    __shared__ float2 wml[NW][32];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hf = lane >> 5, col = lane & 31;
    const uint32_t rep = a.n_head / a.n_kv, rows = a.n * rep;
    // the KV head goes fastest, so that with eight of them an XCD keeps one
    // head's rows in its L2, then the tile, which shares them
    const uint32_t g = blockIdx.x % a.n_kv, tile = blockIdx.x / a.n_kv % a.tiles, sp = blockIdx.x / a.n_kv / a.tiles;
    const uint32_t r0 = 32 * tile + col, r = min(r0, rows - 1);  // lanes past the rows compute a copy
    const uint32_t node = r / rep, h = g * rep + r % rep;
    const uint32_t P = a.len + a.n, nch = (P - 1) / 32 + 1;
    const uint32_t share = (nch + a.S - 1) / a.S, c0 = sp * share, c1 = min(c0 + share, nch);
    const _Float16 *const kb = a.kc + (size_t)g * a.rows * HD;
    const _Float16 *const vb = a.vc + (size_t)g * a.rows * HD;

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
#pragma unroll
            for (int e = 0; e < 8; e++) qm = fmaxf(qm, fabsf(qv[k][e]));
        }
        qm = fmaxf(qm, __shfl_xor(qm, 32, 64));
        int ex;
        (void)frexpf(qm, &ex);
        ex = ex < -60 ? -60 : ex;
        qsc = ldexpf(1.0f, ex) * a.scale * 1.4426950408889634f;  // scores in powers of two
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = ldexpf(qv[k][e], -ex);
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
    float m = -INFINITY, l = 0.f;

    f16x8_t kf[KS];
    auto load_k = [&](uint32_t c) __attribute__((always_inline)) {
        const uint32_t kp = min(32 * c + col, P - 1);  // past the end: a row that is there (not seen)
        const _Float16 *const p = kb + (size_t)kp * HD + 8 * hf;
#pragma unroll
        for (int k = 0; k < KS; k++) kf[k] = *reinterpret_cast<const f16x8_t *>(p + 16 * k);
    };
    if (c0 + wave < c1) load_k(c0 + wave);
    for (uint32_t c = c0 + wave; c < c1; c += NW) {
        // V of position 16 s + 8 (j / 4) + 4 hf + j % 4: slot j of step s
        uint32_t vr[2][8][OT / 2];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t kp = min(32 * c + 16 * s + 8 * (j >> 2) + 4 * hf + (j & 3), P - 1);
                const uint32_t *const p = reinterpret_cast<const uint32_t *>(vb + (size_t)kp * HD) + OT / 2 * col;
                if constexpr (OT == 8) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p);
                    vr[s][j][0] = v.x, vr[s][j][1] = v.y, vr[s][j][2] = v.z, vr[s][j][3] = v.w;
                } else if constexpr (OT == 4) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p);
                    vr[s][j][0] = v.x, vr[s][j][1] = v.y;
                } else {
                    vr[s][j][0] = *p;
                }
            }
        f32x16_t sc;
#pragma unroll
        for (int i = 0; i < 16; i++) sc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], ql[k], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qh[k], sc, 0, 0, 0);
        }
        if (c + NW < c1) load_k(c + NW);
        // the lane's scores are positions 8 (i / 4) + 4 hf + i % 4
        const bool masked = 32 * c + 32 > a.len;
        uint32_t seen = 0xFFFFFFFFu;
        if (masked) seen = seen_bits(a, node, c);
        const uint32_t mine = seen >> (4 * hf);
        float cmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float x = sc[i] * qsc;
            sc[i] = mine >> (8 * (i >> 2) + (i & 3)) & 1 ? x : -INFINITY;
            cmax = fmaxf(cmax, sc[i]);
        }
        cmax = fmaxf(cmax, __shfl_xor(cmax, 32, 64));
        // a row that has seen nothing yet has only -inf: any finite maximum gives zeros
        const float mn = fmaxf(m, cmax) == -INFINITY ? -1e30f : fmaxf(m, cmax);
        const float alpha = __builtin_amdgcn_exp2f(m - mn);
        float ps = 0.f;
        f16x8_t ph[2], pl[2];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(sc[i] - mn);
            ps += p;
            const _Float16 x = (_Float16)p;
            ph[i >> 3][i & 7] = x;
            pl[i >> 3][i & 7] = (_Float16)(p - (float)x);
        }
        ps += __shfl_xor(ps, 32, 64);
        l = l * alpha + ps;
        m = mn;
#pragma unroll
        for (int t = 0; t < OT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] *= alpha;
        // a V that is not finite reaches the rows that see it alone: it is taken
        // out of the product (0 inf is NaN) and added where it is seen
        bool odd = false;
        if (masked) {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int w = 0; w < OT / 2; w++)
                        odd |= (vr[s][j][w] & 0x7C00u) == 0x7C00u || (vr[s][j][w] & 0x7C000000u) == 0x7C000000u;
            odd = __any(odd);
        }
        if (odd) {
            f16x8_t one[2];
#pragma unroll
            for (int i = 0; i < 16; i++)
                one[i >> 3][i & 7] = mine >> (8 * (i >> 2) + (i & 3)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
            for (int t = 0; t < OT; t++) {
                for (int kind = 0; kind < 3; kind++) {  // NaN, inf, -inf
                    f32x16_t n;
#pragma unroll
                    for (int i = 0; i < 16; i++) n[i] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        f16x8_t is;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            uint32_t w = 0;
#pragma unroll
                            for (int i = 0; i < OT / 2; i++) w = i == t / 2 ? vr[s][j][i] : w;
                            const uint32_t b = t & 1 ? w >> 16 : w & 0xFFFFu;
                            const bool hit = kind == 0 ? (b & 0x7FFFu) > 0x7C00u : b == (kind == 1 ? 0x7C00u : 0xFC00u);
                            is[j] = hit ? (_Float16)1.0f : (_Float16)0.0f;
                        }
                        n = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, one[s], n, 0, 0, 0);
                    }
                    const float val = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
                    for (int q = 0; q < OT; q++)
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (q == t && n[i] > 0.f) o[q][i] += val;
                }
            }
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int w = 0; w < OT / 2; w++) {
                        if ((vr[s][j][w] & 0x7C00u) == 0x7C00u) vr[s][j][w] &= 0xFFFF0000u;
                        if ((vr[s][j][w] & 0x7C000000u) == 0x7C000000u) vr[s][j][w] &= 0xFFFFu;
                    }
        }
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int t = 0; t < OT; t++) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    w[j] = __builtin_amdgcn_perm(vr[s][2 * j + 1][t / 2], vr[s][2 * j][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
                const f16x8_t va = __builtin_bit_cast(f16x8_t, w);
                o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[s], o[t], 0, 0, 0);
                o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[s], o[t], 0, 0, 0);
            }
    }
    // the wavefronts' sums over the common maximum, one after another
    if (hf == 0) wml[wave][col] = make_float2(m, l);
    __syncthreads();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, wml[w][col].x);
#pragma unroll
    for (int w = 0; w < NW; w++) {
        const float2 p = wml[w][col];
        if (p.y != 0.f) L += p.y * __builtin_amdgcn_exp2f(p.x - M);
    }
    const float f = l != 0.f ? __builtin_amdgcn_exp2f(m - M) : 0.f;
    for (int w = 0; w < NW; w++) {
        if (wave == (uint32_t)w) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float *const p = osum + col * LD + OT * (8 * (i >> 2) + 4 * hf + (i & 3));
#pragma unroll
                for (int t = 0; t < OT; t++) {
                    const float v = l != 0.f ? o[t][i] * f : 0.f;
                    p[t] = w ? p[t] + v : v;
                }
            }
        }
        __syncthreads();
    }
    // a tile's rows: heads of a node are neighbours in out and in the partials
    if (a.S > 1 && wave == 0 && hf == 0 && r0 < rows) a.ml[((size_t)sp * a.n + node) * a.n_head + h] = make_float2(M, L);
    if (wave == 0 && hf == 0) wml[0][col].x = L != 0.f ? 1.0f / L : 0.f;
    __syncthreads();
    for (uint32_t i = tid; i < 32 * (HD / 4); i += 64 * NW) {
        const uint32_t q = i / (HD / 4), d = 4 * (i % (HD / 4)), row = 32 * tile + q;
        if (row >= rows) break;
        const float4 v = *reinterpret_cast<const float4 *>(osum + q * LD + d);
        const size_t at = ((size_t)(row / rep) * a.n_head + g * rep + row % rep) * HD + d;
        if (a.S > 1) {
            *reinterpret_cast<float4 *>(a.part + (size_t)sp * a.n * a.n_head * HD + at) = v;
        } else {
            const float inv = wml[0][q].x;
            *reinterpret_cast<float4 *>(a.out + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        }
    }
}

// the workgroups' shares of a row joined: thread = 4 elements of a row
__global__ __launch_bounds__(256) void k_tree_merge(AttnTree a, uint32_t hd) {
    const size_t e = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x), N = (size_t)a.n * a.n_head * hd;
    if (e >= N) return;
    const size_t r = e / hd;
    float M = -INFINITY;
    for (uint32_t s = 0; s < a.S; s++) M = fmaxf(M, a.ml[(size_t)s * a.n * a.n_head + r].x);
    float L = 0.f, v[4] = {};
#pragma unroll 4
    for (uint32_t s = 0; s < a.S; s++) {
        const float2 p = a.ml[(size_t)s * a.n * a.n_head + r];
        const float4 x = *reinterpret_cast<const float4 *>(a.part + (size_t)s * N + e);
        if (p.y == 0.f) continue;  // saw nothing
        const float w = __builtin_amdgcn_exp2f(p.x - M);
        L = fmaf(p.y, w, L);
        v[0] = fmaf(w, x.x, v[0]), v[1] = fmaf(w, x.y, v[1]), v[2] = fmaf(w, x.z, v[2]), v[3] = fmaf(w, x.w, v[3]);
    }
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    *reinterpret_cast<float4 *>(a.out + e) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
}

static constexpr uint32_t TREE_NW = 4;

// shares of the positions: about two workgroups per CU, each wavefront at least
// a chunk, and no more partial sums than TREE_WORK holds
uint32_t attn_tree_splits(uint32_t n, uint32_t len, uint32_t n_head, uint32_t n_kv, uint32_t hd) {
    const uint32_t tiles = (n * (n_head / n_kv) + 31) / 32, wgs = tiles * n_kv, chunks = (len + n - 1) / 32 + 1;
    const size_t fit = TREE_WORK / ((size_t)n * n_head * (hd * 4 + 8));
    uint32_t S = (512 + wgs - 1) / wgs;
    S = S < (chunks + TREE_NW - 1) / TREE_NW ? S : (chunks + TREE_NW - 1) / TREE_NW;
    if (S > fit) S = fit ? (uint32_t)fit : 1;
    // no empty share
    const uint32_t share = (chunks + S - 1) / S;
    return (chunks + share - 1) / share;
}

size_t attn_tree_work_bytes(uint32_t n, uint32_t len, uint32_t n_head, uint32_t n_kv, uint32_t hd) {
    const uint32_t S = attn_tree_splits(n, len, n_head, n_kv, hd);
    return S > 1 ? (size_t)S * n * n_head * (hd * 4 + 8) : 0;
}

hipError_t launch_attn_tree(AttnTree a, uint32_t hd, void *work, hipStream_t s) {
    const uint32_t rep = a.n_kv ? a.n_head / a.n_kv : 0;
    if (a.n == 0 || rep == 0 || a.n_head % a.n_kv) return hipErrorInvalidValue;
    a.tiles = (a.n * rep + 31) / 32;
    a.S = attn_tree_splits(a.n, a.len, a.n_head, a.n_kv, hd);
    if (a.S > 1) {
        if (!work) return hipErrorInvalidValue;
        a.part = (float *)work;
        a.ml = (float2 *)(a.part + (size_t)a.S * a.n * a.n_head * hd);
    }
    const dim3 g(a.n_kv * a.tiles * a.S), b(64 * TREE_NW);
    switch (hd) {
    case 64: hipLaunchKernelGGL((k_attn_tree<64, TREE_NW>), g, b, 0, s, a); break;
    case 128: hipLaunchKernelGGL((k_attn_tree<128, TREE_NW>), g, b, 0, s, a); break;
    case 256: hipLaunchKernelGGL((k_attn_tree<256, TREE_NW>), g, b, 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    if (a.S > 1) {
        const size_t q = (size_t)a.n * a.n_head * hd / 4;
        hipLaunchKernelGGL(k_tree_merge, dim3((uint32_t)((q + 255) / 256)), dim3(256), 0, s, a, hd);
    }
    return hipGetLastError();
}

// ---- the walk and the kept rows ---------------------------------------------
// From node 0 down: a node's sampled token is the next token; the walk goes on
// at the first child that drafted it.  out: {length of the walk, its tokens};
// path: its nodes.  One wavefront; a node's parent comes before it, so that
// the walk takes at most n steps.
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
// earlier write has replaced.
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
