// The paged xlns16 KV cache of several sequences: the rotation of the new
// tokens' queries and keys with the stores of their cells, and the attention
// of the new tokens over the cache (include/lnship.h).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lnship.h"
#include "lnship_device.h"
#include "lnship_host.h"

namespace lnship {

// ---- rows and pages -------------------------------------------------------------

// the last s < n with key(s) <= x, key non-decreasing and key(0) <= x
template <class F>
__device__ __forceinline__ int last_at_most(int n, int64_t x, F key) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (key(mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- rope and stores ------------------------------------------------------------

struct store_args {
    lnship_paged_kv kv;
    lnship_paged_store_args a;
    int page_sh;
};

// One thread per element of a row's heads (query, key, value heads in turn);
// what a thread reads and converts alone is as in lnship16_rope and
// lnship16_store_kv.
__global__ __launch_bounds__(k_block) void k_store_paged(store_args s, dev_tables T, unsigned long long *err) {
    const fmt16 F{T};
    const lnship_paged_kv &kv = s.kv;
    const lnship_paged_store_args &a = s.a;
    const int64_t t = blockIdx.x, hd = kv.head_dim;
    const int n_seq = (int)kv.n_seq;
    if (t < kv.q_start[0] || t >= kv.q_start[n_seq]) return;
    const int sq = last_at_most(n_seq, t, [&](int i) { return kv.q_start[i]; });
    const int64_t p = (int64_t)kv.kv_len[sq] - kv.q_start[sq + 1] + t;
    const int nd = a.rope_n_dims;
    if (p < 0 || p >> s.page_sh >= kv.table_ld || (nd > 0 && p >= a.n_pos)) {
        if (blockIdx.y == 0 && threadIdx.x == 0) index_fault(err, p);
        return;
    }
    const int64_t id = kv.table[sq * kv.table_ld + (p >> s.page_sh)], c = p & (kv.page - 1);
    const bool paged = id >= 0 && id < kv.n_pages;
    if (!paged && blockIdx.y == 0 && threadIdx.x == 0) index_fault(err, id);
    const float *cs = nd > 0 ? a.cos_sin + p * nd : nullptr;
    const int64_t nq = a.n_head * hd, nk = kv.n_head_kv * hd;
    for (int64_t i = (int64_t)blockIdx.y * k_block + threadIdx.x; i < nq + 2 * nk; i += (int64_t)gridDim.y * k_block) {
        const int part = i < nq ? 0 : i < nq + nk ? 1 : 2;
        const int64_t e = part == 0 ? i : part == 1 ? i - nq : i - nq - nk;
        const int64_t h = e / hd, d = e - h * hd;
        const float *x = part == 0 ? a.q + t * a.q_ld : part == 1 ? a.k + t * a.k_ld : a.v + t * a.v_ld;
        x += h * hd;
        float v = x[d];
        if (part < 2 && nd > 0) {
            if (d < nd) {
                const int64_t half = nd / 2, j = a.neox ? d % half : d / 2;
                int64_t i0, i1;
                uint32_t r0, r1;
                rope_pair(F, x, j, nd, a.neox, cs, i0, i1, r0, r1);
                v = F.to(d == i0 ? r0 : r1);
            } else {
                v = F.to(F.from(v));
            }
        }
        if (part == 0) {
            a.q_dst[t * a.q_dst_ld + e] = v;
        } else if (paged) {
            const int64_t base = (id * kv.n_head_kv + h) * kv.page * hd;
            uint16_t *o = part == 1 ? kv.k_pages + base + ((d >> 3) * kv.page + c) * 8 + (d & 7)
                                    : kv.v_pages + base + ((c >> 3) * hd + d) * 8 + (c & 7);
            *o = (uint16_t)F.from(__half2float(__float2half_rn(v)));
        }
    }
}

// ---- attention --------------------------------------------------------------------

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

struct attn_paged_args {
    lnship_paged_kv kv;
    const float *q;
    float *dst;
    int64_t q_ld, dst_ld, window;
    float scale;          // times log2 e
    int n_head, rep, page_sh, splits;
    float *work;          // [splits][ntok][n_head] rows of head_dim sums, maximum and total
};

constexpr int k_lo_sh = 11;             // the low halves are scaled by 2^11
constexpr float k_lo = 2048.0f, k_lo_inv = 1.0f / 2048.0f;
constexpr float k_p_scale = 16384.0f;   // of the weights as halves

// x, y to a pair of halves, and what the rounding leaves, times 2^11, to
// another: together 22 bits of each
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const half2v h = {(_Float16)x, (_Float16)y};
    const half2v l = {(_Float16)((x - (float)h[0]) * k_lo), (_Float16)((y - (float)h[1]) * k_lo)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// Two xlns16 codes in a word to the split halves of their values.  The log
// field goes into the mantissa of 2^23 + log, one FMA makes it the exponent;
// 2^11 times the value stays within F32 and the split needs no other product.
// Log 0 (zero) becomes 2^-117, which rounds to zero in both halves.
__device__ __forceinline__ void decode2(uint32_t w, uint32_t &hi, uint32_t &lo) {
    constexpr uint32_t magic = 0x4b000000u, top = 0x47ffu;   // 2^23; the largest log of a half
    const uint32_t l0 = min(w & k16_logmask, top), l1 = min((w >> 16) & k16_logmask, top);
    constexpr float off = -(8388608.0f / 128 + 128 - k_lo_sh);
    const float x0 = __builtin_amdgcn_exp2f(fmaf(__uint_as_float(magic | l0), 1.0f / 128, off));
    const float x1 = __builtin_amdgcn_exp2f(fmaf(__uint_as_float(magic | l1), 1.0f / 128, off));
    const half2v h = {(_Float16)(x0 * k_lo_inv), (_Float16)(x1 * k_lo_inv)};
    const half2v l = {(_Float16)fmaf((float)h[0], -k_lo, x0), (_Float16)fmaf((float)h[1], -k_lo, x1)};
    const uint32_t sg = w & (k16_sign << 16 | k16_sign);
    hi = __builtin_bit_cast(uint32_t, h) ^ sg;
    lo = __builtin_bit_cast(uint32_t, l) ^ sg;
}

union frag {   // a lane's eight halves of a matrix operand
    uint4 w;
    uint32_t u[4];
    half8 h;
};

__device__ __forceinline__ void decode8(uint4 c, frag &hi, frag &lo) {
    decode2(c.x, hi.u[0], lo.u[0]);
    decode2(c.y, hi.u[1], lo.u[1]);
    decode2(c.z, hi.u[2], lo.u[2]);
    decode2(c.w, hi.u[3], lo.u[3]);
}

__device__ __forceinline__ float4v mma(const frag &a, const frag &b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}

// A wave takes 16 rows (token and head of one kv head's group) and, of their
// visible cells, every fourth block of 32; the four waves of a workgroup and
// the workgroups of a split are joined by their maxima.  Scores are formed
// transposed, S^T = K Q^T, with the cells dealt to the rows of two 16 x 16
// products so that a lane's eight scores are eight neighbouring cells of one
// row: as such they are the operand of O^T = V^T P^T, and both caches' layouts
// give a lane's share of K and V in 16-byte loads.
template <int NB>   // 32-wide groups of head_dim
__global__ __launch_bounds__(256) void k_attn_paged(attn_paged_args a, unsigned long long *err) {
    const lnship_paged_kv &kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int rep = a.rep, kvh = blockIdx.y, split = blockIdx.z, hd = (int)kv.head_dim;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ float s_o[16][NB * 32 + 1];

    // the tile's sequence: sequence s's tiles start at q_start[s] rep / 16 + s
    const int64_t tile = blockIdx.x;
    const int sq = last_at_most((int)kv.n_seq, tile,
                                [&](int i) { return (int64_t)max(kv.q_start[i], 0) * rep / 16 + i; });
    const int64_t t0 = max(kv.q_start[sq], 0), t1 = min((int64_t)kv.q_start[sq + 1], kv.ntok);
    const int64_t r0 = (tile - (t0 * rep / 16 + sq)) * 16, rows = (t1 - t0) * rep;
    if (r0 < 0 || r0 >= rows) return;
    const int64_t pos0 = (int64_t)kv.kv_len[sq] - kv.q_start[sq + 1] + t0;
    const int64_t cells = kv.table_ld << a.page_sh;
    const int64_t last = pos0 + (min(r0 + 16, rows) - 1) / rep, first = pos0 + r0 / rep;
    if (last >= cells && threadIdx.x == 0) index_fault(err, last);
    const int64_t c1 = min(last + 1, cells);
    const int64_t c0 = a.window > 0 ? max((int64_t)0, first - a.window + 1) & ~(int64_t)31 : 0;
    // this split's blocks of 32 cells, at least 8 a split
    const int64_t blocks = c1 > c0 ? (c1 - c0 + 31) / 32 : 0;
    const int64_t per = max((blocks + a.splits - 1) / a.splits, (int64_t)8);
    const int64_t b0 = split * per, b1 = min(b0 + per, blocks);
    if (split > 0 && b0 >= blocks) return;

    // the lane's row
    const int64_t row = r0 + n;
    const bool have = row < rows;
    const int64_t tok = t0 + (have ? row / rep : 0);
    const int head = kvh * rep + (have ? (int)(row % rep) : 0);
    const int64_t pos = pos0 + tok - t0;
    const int64_t lo_cell = a.window > 0 ? pos - a.window : -1;   // cells at and below are hidden

    // the queries as halves, scaled by the row's largest to at most 2
    frag qh[NB], ql[NB];
    float qs;
    {
        float x[NB][8], mx = 0.0f;
        const float *q = a.q + tok * a.q_ld + (int64_t)head * hd;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int d = b * 32 + g * 8 + j;
                x[b][j] = have && d < hd ? q[d] : 0.0f;
                mx = fmaxf(mx, fabsf(x[b][j]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int e = (int)(f32_bits(mx) >> 23) - 127;   // -127 for zeros
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                split2(ldexpf(x[b][j], -e), ldexpf(x[b][j + 1], -e), qh[b].u[j / 2], ql[b].u[j / 2]);
        qs = ldexpf(a.scale, e);
    }

    float4v o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) o[i] = float4v{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    const int32_t *table = kv.table + sq * kv.table_ld;
    for (int64_t b = b0 + wave; b < b1; b += 4) {
        const int64_t cb = c0 + b * 32;
        // the lane's cells: as a row of K^T's products, and of its eight scores
        int64_t kpg = -1, vpg = -1;
        const int64_t kc = cb + 8 * (n >> 2), vc = cb + 8 * g;
        if (kc < c1) kpg = table[kc >> a.page_sh];
        if (vc < c1) vpg = table[vc >> a.page_sh];
        const bool kok = kc < c1 && kpg >= 0 && kpg < kv.n_pages, vok = vc < c1 && vpg >= 0 && vpg < kv.n_pages;
        if (vc < c1 && !vok) index_fault(err, vpg);
        const uint4 zero = make_uint4(0, 0, 0, 0);
        float4v sh[2], sx[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            sh[t] = sx[t] = float4v{0, 0, 0, 0};
            const int64_t cell = (kc & (kv.page - 1)) + 4 * t + (n & 3);
            const uint16_t *k = kv.k_pages + ((kok ? kpg : 0) * kv.n_head_kv + kvh) * kv.page * hd;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                uint4 c = zero;
                if (kok && i * 32 + g * 8 < hd)
                    c = *reinterpret_cast<const uint4 *>(k + ((int64_t)(i * 4 + g) * kv.page + cell) * 8);
                frag kh, kl;
                decode8(c, kh, kl);
                sh[t] = mma(kh, qh[i], sh[t]);
                sx[t] = mma(kl, qh[i], sx[t]);
                sx[t] = mma(kh, ql[i], sx[t]);
            }
        }
        float s[8], mb = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int64_t cell = vc + j;
            s[j] = (sh[j >> 2][j & 3] + k_lo_inv * sx[j >> 2][j & 3]) * qs;
            if (!vok || cell > pos || cell <= lo_cell) s[j] = -INFINITY;
            mb = fmaxf(mb, s[j]);
        }
        mb = fmaxf(mb, __shfl_xor(mb, 16));
        mb = fmaxf(mb, __shfl_xor(mb, 32));
        const float mn = fmaxf(m, mb), ms = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ms);
        m = mn;
        float p[8];
        frag ph, pl, pc;
        l *= alpha;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(s[j] - ms);
            l += p[j];
        }
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float x = p[j] * k_p_scale, y = p[j + 1] * k_p_scale;
            const half2v h = {(_Float16)x, (_Float16)y};
            const half2v r = {(_Float16)(x - (float)h[0]), (_Float16)(y - (float)h[1])};
            const half2v f = {(_Float16)k_lo_inv, (_Float16)k_lo_inv};
            const half2v c = h * f;
            ph.u[j / 2] = __builtin_bit_cast(uint32_t, h);
            pl.u[j / 2] = __builtin_bit_cast(uint32_t, r);
            pc.u[j / 2] = __builtin_bit_cast(uint32_t, c);
        }
        const uint16_t *v = kv.v_pages + ((vok ? vpg : 0) * kv.n_head_kv + kvh) * kv.page * hd +
                            ((vc & (kv.page - 1)) >> 3) * hd * 8;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            uint4 c = zero;
            if (vok && i * 16 + n < hd) c = *reinterpret_cast<const uint4 *>(v + (i * 16 + n) * 8);
            frag vh, vl;
            decode8(c, vh, vl);
            o[i] *= alpha;
            o[i] = mma(vh, ph, o[i]);
            o[i] = mma(vh, pl, o[i]);
            o[i] = mma(vl, pc, o[i]);
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' parts joined, in the waves' order
    if (g == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(s_m[0][n], s_m[1][n]), fmaxf(s_m[2][n], s_m[3][n]));
    const float Ms = M == -INFINITY ? 0.0f : M;
    const float f = __builtin_amdgcn_exp2f(m - Ms) * (1.0f / k_p_scale);
    for (int w = 0; w < 4; w++) {
        if (wave == w) {
#pragma unroll
            for (int i = 0; i < 2 * NB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float &x = s_o[n][i * 16 + g * 4 + j];
                    x = (w ? x : 0.0f) + o[i][j] * f;
                }
        }
        __syncthreads();
    }
    // a row's elements, on 16 threads
    const int rr = threadIdx.x >> 4;
    const int64_t row2 = r0 + rr;
    if (row2 >= rows) return;
    const int64_t tok2 = t0 + row2 / rep;
    const int head2 = kvh * rep + (int)(row2 % rep);
    float M2 = -INFINITY, L2 = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) M2 = fmaxf(M2, s_m[w][rr]);
    const float Ms2 = M2 == -INFINITY ? 0.0f : M2;
#pragma unroll
    for (int w = 0; w < 4; w++) L2 += s_l[w][rr] * __builtin_amdgcn_exp2f(s_m[w][rr] - Ms2);
    if (a.splits == 1) {
        const float inv = M2 == -INFINITY ? 0.0f : 1.0f / L2;
        float *dst = a.dst + tok2 * a.dst_ld + (int64_t)head2 * hd;
        for (int d = threadIdx.x & 15; d < hd; d += 16) dst[d] = s_o[rr][d] * inv;
    } else {
        float *dst = a.work + ((split * kv.ntok + tok2) * a.n_head + head2) * (hd + 2);
        for (int d = threadIdx.x & 15; d < hd; d += 16) dst[d] = s_o[rr][d];
        if ((threadIdx.x & 15) == 0) {
            dst[hd] = M2;
            dst[hd + 1] = L2;
        }
    }
}

// The splits' parts of a row joined, in the splits' order.
__global__ __launch_bounds__(64) void k_attn_paged_join(attn_paged_args a) {
    const lnship_paged_kv &kv = a.kv;
    const int64_t tok = blockIdx.x;
    const int head = blockIdx.y, hd = (int)kv.head_dim, n_seq = (int)kv.n_seq;
    if (tok < kv.q_start[0] || tok >= kv.q_start[n_seq]) return;
    const int sq = last_at_most(n_seq, tok, [&](int i) { return kv.q_start[i]; });
    const int64_t t0 = max(kv.q_start[sq], 0), t1 = min((int64_t)kv.q_start[sq + 1], kv.ntok);
    const int64_t pos0 = (int64_t)kv.kv_len[sq] - kv.q_start[sq + 1] + t0;
    // the splits that the row's tile had, as k_attn_paged finds them
    const int64_t rows = (t1 - t0) * a.rep, r0 = ((tok - t0) * a.rep + head % a.rep) & ~(int64_t)15;
    const int64_t last = pos0 + (min(r0 + 16, rows) - 1) / a.rep, first = pos0 + r0 / a.rep;
    const int64_t c1 = min(last + 1, kv.table_ld << a.page_sh);
    const int64_t c0 = a.window > 0 ? max((int64_t)0, first - a.window + 1) & ~(int64_t)31 : 0;
    const int64_t blocks = c1 > c0 ? (c1 - c0 + 31) / 32 : 0;
    const int64_t per = max((blocks + a.splits - 1) / a.splits, (int64_t)8);
    const int used = (int)max((blocks + per - 1) / per, (int64_t)1);
    const int64_t step = kv.ntok * a.n_head * (hd + 2);
    const float *w = a.work + (tok * a.n_head + head) * (hd + 2);
    float M = -INFINITY;
    for (int i = 0; i < used; i++) M = fmaxf(M, w[i * step + hd]);
    const float Ms = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    for (int i = 0; i < used; i++) L += w[i * step + hd + 1] * __builtin_amdgcn_exp2f(w[i * step + hd] - Ms);
    const float inv = M == -INFINITY ? 0.0f : 1.0f / L;
    float *dst = a.dst + tok * a.dst_ld + (int64_t)head * hd;
    for (int d = threadIdx.x; d < hd; d += 64) {
        float s = 0.0f;
        for (int i = 0; i < used; i++) s += w[i * step + d] * __builtin_amdgcn_exp2f(w[i * step + hd] - Ms);
        dst[d] = s * inv;
    }
}

// ---- host -----------------------------------------------------------------------

// sizes (and, with ptrs, pointers) of a paged cache and its batch
static int check_paged(const lnship_paged_kv *kv, bool ptrs) {
    if (!kv || kv->ntok < 0 || kv->n_seq < 0 || kv->n_head_kv < 1 || kv->n_pages < 0 || kv->table_ld < 0)
        return fail(LNSHIP_EINVAL, "paged cache: bad shape%s");
    if (kv->page < 16 || kv->page > 256 || (kv->page & (kv->page - 1)))
        return fail(LNSHIP_EINVAL, "paged cache: page not a power of two from 16 to 256%s");
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
        return fail(LNSHIP_EINVAL, "paged cache: head_dim not a multiple of 8 up to 256%s");
    // (a grid's threads along x are counted in 32 bits)
    if (kv->ntok > 0xffffff || kv->n_seq > 0x7fffff || kv->n_head_kv > 65535 || kv->n_pages > 0x7fffffff ||
        kv->table_ld > 0x7fffffff / kv->page)
        return fail(LNSHIP_ERANGE, "paged cache: too large%s");
    if (ptrs && kv->ntok && kv->n_seq) {
        if (!kv->k_pages || !kv->v_pages || !kv->q_start || !kv->kv_len || (!kv->table && kv->table_ld))
            return fail(LNSHIP_EINVAL, "paged cache: null pointer%s");
        if (((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15)
            return fail(LNSHIP_EINVAL, "paged cache: pages not 16-byte aligned%s");
    }
    return 0;
}

static int log2_of(int64_t page) {
    int sh = 0;
    while ((int64_t)1 << sh < page) sh++;
    return sh;
}

static int64_t attn_tiles(const lnship_paged_kv *kv, int64_t rep) { return kv->ntok * rep / 16 + kv->n_seq; }

// Parts that a row's cells are split into: where there are few tiles, as many
// as give every CU two workgroups, each of at least 8 blocks of 32 cells.
static int attn_splits(const lnship_paged_kv *kv, int64_t rep, int cus) {
    const int64_t wgs = std::max<int64_t>(1, attn_tiles(kv, rep) * kv->n_head_kv);
    const int64_t most = (kv->table_ld * kv->page + 255) / 256;
    return (int)std::max<int64_t>(1, std::min<int64_t>({(2 * cus + wgs - 1) / wgs, most, 256}));
}

static int64_t attn_work(const lnship_paged_kv *kv, int64_t n_head, int splits) {
    return splits > 1 ? (int64_t)splits * kv->ntok * n_head * (kv->head_dim + 2) * 4 : 0;
}

}  // namespace lnship

using namespace lnship;

extern "C" {

int lnship16_rope_store_kv_paged(const lnship_paged_kv *kv, const lnship_paged_store_args *a, void *stream) {
    if (int rc = check_paged(kv, true)) return rc;
    if (!a || a->n_head < 0 || a->rope_n_dims < 0 || a->rope_n_dims % 2 || a->rope_n_dims > kv->head_dim)
        return fail(LNSHIP_EINVAL, "rope_store_kv_paged: bad shape%s");
    store_args s{*kv, *a, log2_of(kv->page)};
    const int64_t nq = a->n_head * kv->head_dim, nk = kv->n_head_kv * kv->head_dim;
    if (!s.a.q_dst_ld) s.a.q_dst_ld = nq;
    if (nq > 0x7fffffff || a->q_ld < (a->n_head ? nq : 0) || a->k_ld < nk || a->v_ld < nk || s.a.q_dst_ld < nq || a->n_pos < 0)
        return fail(LNSHIP_EINVAL, "rope_store_kv_paged: bad shape%s");
    if (kv->ntok == 0 || kv->n_seq == 0) return 0;
    if (!a->k || !a->v || (a->n_head && (!a->q || !a->q_dst)) || (a->rope_n_dims && !a->cos_sin))
        return fail(LNSHIP_EINVAL, "rope_store_kv_paged: null pointer%s");
    device_state *st = state();
    if (!st) return LNSHIP_ENOINIT;
    const int64_t y = std::min<int64_t>((nq + 2 * nk + k_block - 1) / k_block, 65535);
    hipLaunchKernelGGL(k_store_paged, dim3((unsigned)kv->ntok, (unsigned)y), dim3(k_block), 0, (hipStream_t)stream, s,
                       st->T, st->index_err);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

int64_t lnship16_attn_paged_work(const lnship_paged_kv *kv, int64_t n_head) {
    if (int rc = check_paged(kv, false)) return rc;
    if (n_head < 1 || n_head % kv->n_head_kv || n_head > 65535)
        return fail(LNSHIP_EINVAL, "attn_paged: n_head not a multiple of n_head_kv%s");
    device_state *st = state();
    if (!st) return LNSHIP_ENOINIT;
    return attn_work(kv, n_head, attn_splits(kv, n_head / kv->n_head_kv, st->cus));
}

int lnship16_attn_paged(const lnship_paged_kv *kv, const lnship_paged_attn_args *a, void *stream) {
    if (int rc = check_paged(kv, true)) return rc;
    if (!a || a->n_head < 1 || a->n_head % kv->n_head_kv || a->n_head > 65535 || a->window < 0)
        return fail(LNSHIP_EINVAL, "attn_paged: bad shape%s");
    const int64_t nq = a->n_head * kv->head_dim;
    const int64_t q_ld = a->q_ld ? a->q_ld : nq, dst_ld = a->dst_ld ? a->dst_ld : nq;
    if (q_ld < nq || dst_ld < nq) return fail(LNSHIP_EINVAL, "attn_paged: bad shape%s");
    if (kv->ntok == 0 || kv->n_seq == 0) return 0;
    if (!a->q || !a->dst) return fail(LNSHIP_EINVAL, "attn_paged: null pointer%s");
    device_state *st = state();
    if (!st) return LNSHIP_ENOINIT;
    const int64_t rep = a->n_head / kv->n_head_kv;
    const int splits = attn_splits(kv, rep, st->cus);
    const int64_t need = attn_work(kv, a->n_head, splits), tiles = attn_tiles(kv, rep);
    if (need && (!a->work || a->work_bytes < (size_t)need || ((uintptr_t)a->work & 15)))
        return fail(LNSHIP_EINVAL, "attn_paged: work smaller than lnship16_attn_paged_work or not aligned%s");
    if (tiles > 0xffffff) return fail(LNSHIP_ERANGE, "attn_paged: grid too large%s");
    attn_paged_args m{*kv, a->q, a->dst, q_ld, dst_ld, std::min<int64_t>(a->window, (int64_t)1 << 40),
                      a->scale * 1.44269504088896341f, (int)a->n_head, (int)rep, log2_of(kv->page), splits,
                      (float *)a->work};
    const dim3 grid((unsigned)tiles, (unsigned)kv->n_head_kv, (unsigned)splits), block(256);
    hipStream_t s = (hipStream_t)stream;
    switch ((kv->head_dim + 31) / 32) {
#define LNSHIP_ATTN(NB) \
    case NB: hipLaunchKernelGGL(k_attn_paged<NB>, grid, block, 0, s, m, st->index_err); break
        LNSHIP_ATTN(1);
        LNSHIP_ATTN(2);
        LNSHIP_ATTN(3);
        LNSHIP_ATTN(4);
        LNSHIP_ATTN(5);
        LNSHIP_ATTN(6);
        LNSHIP_ATTN(7);
        default: hipLaunchKernelGGL(k_attn_paged<8>, grid, block, 0, s, m, st->index_err);
#undef LNSHIP_ATTN
    }
    LNSHIP_HIP(hipGetLastError());
    if (splits > 1) {
        hipLaunchKernelGGL(k_attn_paged_join, dim3((unsigned)kv->ntok, (unsigned)a->n_head), dim3(64), 0, s, m);
        LNSHIP_HIP(hipGetLastError());
    }
    return 0;
}

}  // extern "C"
