// The paged xlns16 KV cache of several sequences: the rotation of the new
// tokens' queries and keys with the stores of their cells, and the attention
// of the new tokens over the cache (include/lnship.h).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

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

// The same by a whole wave, 64 keys a round: a round takes as long as a step
// above, and up to 64 sequences take one.
template <class F>
__device__ __forceinline__ int wave_last_at_most(int n, int x, F key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 63) >> 6, i = lane * step;
        const uint64_t in = __ballot(i < len && key(lo + min(i, len - 1)) <= x);
        const int last = max(__popcll(in) - 1, 0) * step;   // (keys rise: the lanes in are the first ones)
        lo += last;
        len = min(step, len - last);
    }
    return lo;
}

// ---- rope and stores ------------------------------------------------------------

struct store_args {
    lnship_paged_kv kv;
    lnship_paged_store_args a;
    int page_sh;
};

// One thread per rotated pair, or other element, of a row's heads (query, key,
// value heads in turn), as in lnship16_rope and lnship16_store_kv: a thread
// writes what it alone has read, so that q_dst may be q.
__global__ __launch_bounds__(k_block) void k_store_paged(store_args s, dev_tables T, unsigned long long *err) {
    const fmt16 F{T};
    const lnship_paged_kv &kv = s.kv;
    const lnship_paged_store_args &a = s.a;
    const int64_t t = blockIdx.x, hd = kv.head_dim;
    const int n_seq = (int)kv.n_seq;
    if (t < kv.q_start[0] || t >= kv.q_start[n_seq]) return;
    const int sq = wave_last_at_most(n_seq, (int)t, [&](int i) { return kv.q_start[i]; });
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
    const int64_t pairs = nd / 2, of_head = hd - pairs;   // items of a query or key head
    const int64_t nq = a.n_head * of_head, nk = kv.n_head_kv * of_head, nv = kv.n_head_kv * hd;
    for (int64_t i = (int64_t)blockIdx.y * k_block + threadIdx.x; i < nq + nk + nv; i += (int64_t)gridDim.y * k_block) {
        const int part = i < nq ? 0 : i < nq + nk ? 1 : 2;
        const int64_t e = part == 0 ? i : part == 1 ? i - nq : i - nq - nk, items = part < 2 ? of_head : hd;
        const int64_t h = e / items, j = e - h * items;
        const float *x = part == 0 ? a.q + t * a.q_ld : part == 1 ? a.k + t * a.k_ld : a.v + t * a.v_ld;
        x += h * hd;
        // the thread's element, or pair (all loads before the stores)
        const bool pair = part < 2 && j < pairs;
        int64_t d0 = part < 2 ? j + pairs : j, d1 = d0;
        float v0, v1;
        if (pair) {
            uint32_t r0, r1;
            rope_pair(F, x, j, nd, a.neox, cs, d0, d1, r0, r1);
            v0 = F.to(r0);
            v1 = F.to(r1);
        } else {
            v0 = v1 = part < 2 && nd > 0 ? F.to(F.from(x[d0])) : x[d0];
        }
        if (part == 0) {
            float *o = a.q_dst + t * a.q_dst_ld + h * hd;
            o[d0] = v0;
            if (pair) o[d1] = v1;
        } else if (paged) {
            const uint16_t c0 = (uint16_t)F.from(__half2float(__float2half_rn(v0)));
            const uint16_t c1 = (uint16_t)F.from(__half2float(__float2half_rn(v1)));
            uint16_t *o = (part == 1 ? kv.k_pages : kv.v_pages) + (id * kv.n_head_kv + h) * kv.page * hd;
            auto at = [&](int64_t d) { return part == 1 ? ((d >> 3) * kv.page + c) * 8 + (d & 7) : ((c >> 3) * hd + d) * 8 + (c & 7); };
            o[at(d0)] = c0;
            if (pair) o[at(d1)] = c1;
        }
    }
}

// The rotation of a pair of codes by cs, the cosine's code and above it the sine's:
// y0 = x0 cos - x1 sin, y1 = x0 sin + x1 cos, as x16_mul and x16_add_g form them.
// Of the two sums exactly one is of two addends alike in sign.
__device__ __forceinline__ void rotate_pair(const int16_t *g, uint32_t x0, uint32_t x1, uint32_t cs, uint32_t &y0, uint32_t &y1) {
    const int l0 = x0 & k16_logmask, l1 = x1 & k16_logmask, lc = cs & k16_logmask, ls = cs >> 16 & k16_logmask;
    auto in_range = [](int l) { return min(max(l, 0), (int)k16_logmask); };
    auto sum = [&](int p, int q, uint32_t sp, uint32_t sq, bool differ) {
        const int most = max(p, q), d = most - min(p, q);
        const int l = in_range(most + g[min(d, k16_esszer + 1) + (differ ? k16_gauss_n : 0)]);
        const uint32_t r = ((p > q ? sp : sq) & k16_sign) | (uint32_t)l;
        return (d == 0 && differ) ? 0u : r;
    };
    constexpr int one = (int)k16_one;
    const uint32_t s0 = x0 ^ cs, s1 = x1 ^ cs >> 16;   // (bit 15)
    const bool alike = (s0 ^ s1) & k16_sign;           // of x0 cos and -x1 sin
    y0 = sum(in_range(l0 + lc - one), in_range(l1 + ls - one), s0, ~s1, !alike);
    y1 = sum(in_range(l0 + ls - one), in_range(l1 + lc - one), x0 ^ cs >> 16, x1 ^ cs, alike);
}

// The codes of a rotated key through F32 and half and back, for a code whose
// value is a normal half: its exponent, and of its fraction one of two tables
// of 128 (below 1 the conversion's truncation is upward).  Any other code takes
// the way through the tables in memory.
struct half_codes {
    const int16_t *t;   // LDS: [0, 128) below 1, [128, 256) from 1 on; the new fraction (up to 128)
    const dev_tables &T;
    __device__ __forceinline__ uint32_t slow(uint32_t c) const {
        return x16_from_f32(T.cvt16, __half2float(__float2half_rn(T.rev16[c])));
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t c) const {
        const uint32_t l = c & k16_logmask, e = l >> 7;
        uint32_t r = (c & (k16_sign | 0x7f80u)) + (uint32_t)(int32_t)t[(l & 127u) + (e < 128u ? 0u : 128u)];
        if (__builtin_expect(e - 114u >= 29u, 0)) r = slow(c);   // below 2^-14, or 2^15 and more
        return r;
    }
};

// The F32 value of a code: those of 2^-8 to 2^8 from LDS.
constexpr int k_rev_binades = 16, k_rev_lds = k_rev_binades * 128;
struct rev16_lds {
    const float *t;
    const float *rev;
    __device__ __forceinline__ float operator()(uint32_t c) const {
        const uint32_t i = (c & k16_logmask) - (k16_one - k_rev_lds / 2);
        float v = t[min(i, (uint32_t)k_rev_lds - 1u)];
        v = __uint_as_float(f32_bits(v) | (c & k16_sign) << 16);
        if (__builtin_expect(i >= (uint32_t)k_rev_lds, 0)) v = rev[c];
        return v;
    }
};

constexpr int k_store_rows = 8;   // rows of a workgroup at most

// Many rows, in 16-byte loads: a thread rotates four pairs (or converts eight
// dims behind the rotated ones) of a head, or stores four dims of a value; a
// workgroup has one row or eight, threads beside each other taking the rows of
// one item, whose cells then fill cache lines in one store.  The conversions, the
// Gaussian logs and the decoded values come from tables in LDS: from memory each
// is a gather that costs a cache line a lane.  A row's cosines and sines are
// converted once for all heads.  Bound by VALU issue, 137 instructions a pair with
// its conversions, its value or cell and its share of the values' stores (counted:
// 69 % of the kernel's cycles, 87 % of those in which a CU has work; the rest are the
// tables and the end): 11414 rows of 32 heads of 64 on 8 in 70 us, 3.7 TB/s of what is
// read and written.  With rows spread over all XCDs it took 1.2 times as long (the
// caches' lines are then written in parts), with registers for six waves a SIMD in
// place of eight 1.04 times.
template <bool NEOX>
__global__ __launch_bounds__(k_block, 8) void k_store_paged_rows(store_args s, int row_sh, dev_tables T,
                                                              unsigned long long *err) {
    __shared__ uint16_t s_cvt[k_cvt_lds];
    __shared__ alignas(16) int16_t s_g[2 * k16_gauss_n];
    __shared__ int16_t s_half[256];
    __shared__ float s_rev[k_rev_lds];
    __shared__ int s_pos[k_store_rows], s_page[k_store_rows];
    __shared__ alignas(16) uint16_t s_cs[k_store_rows * 256];
    const lnship_paged_kv &kv = s.kv;
    const lnship_paged_store_args &a = s.a;
    const int tid = threadIdx.x, hd = (int)kv.head_dim, nd = a.rope_n_dims, page = (int)kv.page;
    const int n_head = (int)a.n_head, n_head_kv = (int)kv.n_head_kv, n_seq = (int)kv.n_seq;
    // rows side by side on one XCD: their cells share cache lines
    const uint32_t of_xcd = (gridDim.x + 7) / 8, wg = blockIdx.x % 8 * of_xcd + blockIdx.x / 8;
    const int64_t t0 = (int64_t)wg << row_sh;
    const int rows = (int)min((int64_t)1 << row_sh, kv.ntok - t0);
    if (rows <= 0) return;
    if (tid < rows) {
        const int64_t t = t0 + tid;
        int pos = -1, id = -1;
        if (t >= kv.q_start[0] && t < kv.q_start[n_seq]) {
            // single tokens: row t is sequence t's
            int sq = (int)min(t, (int64_t)n_seq - 1);
            if (kv.q_start[sq] > t || kv.q_start[sq + 1] <= t)
                sq = last_at_most(n_seq, t, [&](int i) { return kv.q_start[i]; });
            const int64_t p = (int64_t)kv.kv_len[sq] - kv.q_start[sq + 1] + t;
            if (p < 0 || p >> s.page_sh >= kv.table_ld || p >= a.n_pos) {
                index_fault(err, p);
            } else {
                pos = (int)p;
                id = kv.table[sq * kv.table_ld + (p >> s.page_sh)];
                if (id < 0 || id >= kv.n_pages) {
                    index_fault(err, id);
                    id = -1;
                }
            }
        }
        s_pos[tid] = pos;
        s_page[tid] = id;
    }
    const cvt16_lds C = stage_cvt16(T.cvt16, s_cvt);
    for (int i = tid; i < k16_gauss_n; i += k_block)
        reinterpret_cast<uint32_t *>(s_g)[i] = reinterpret_cast<const uint32_t *>(T.gauss16)[i];
    for (int i = tid; i < k_rev_lds; i += k_block) s_rev[i] = T.rev16[k16_one - k_rev_lds / 2 + i];
    const half_codes H{s_half, T};
    for (int i = tid; i < 256; i += k_block) s_half[i] = (int16_t)(H.slow(k16_one - 128 + i) - (k16_one + (i & 128) - 128));
    const rev16_lds V{s_rev, T.rev16};
    __syncthreads();
    // a row's cosines and sines, once for all heads
    for (int i = tid * 4; i < rows * nd; i += k_block * 4) {
        const int r = (int)((uint32_t)i / (uint32_t)nd);
        if (s_pos[r] < 0) continue;
        const float4 u = *reinterpret_cast<const float4 *>(a.cos_sin + (int64_t)s_pos[r] * nd + (i - r * nd));
        const float w[4] = {u.x, u.y, u.z, u.w};
        uint32_t z[4];
#pragma unroll
        for (int j = 0; j < 4; j++) z[j] = C(w[j]);
        *reinterpret_cast<uint2 *>(&s_cs[i]) = make_uint2(z[0] | z[1] << 16, z[2] | z[3] << 16);
    }
    __syncthreads();

    const int eighths = hd >> 3, rot_q = n_head * eighths, rot = rot_q + n_head_kv * eighths;
    const int nk = n_head_kv * hd, span = 64 >> row_sh, per = rot + (nk + 4 * span - 1) / (4 * span) * span;
    const int64_t head_codes = (int64_t)page * hd;
    for (int i = (int)(blockIdx.y * k_block) + tid; i < per << row_sh; i += (int)(gridDim.y * k_block)) {
        const int r = i & ((1 << row_sh) - 1), e = i >> row_sh;
        if (r >= rows) continue;
        const int pos = s_pos[r], id = s_page[r];
        const int64_t t = t0 + r;
        if (pos >= 0) {
            const int c = pos & (page - 1);
            if (e < rot) {
                const bool key = e >= rot_q;
                const int f = key ? e - rot_q : e, h = (int)((uint32_t)f / (uint32_t)eighths), o = f - h * eighths;
                const float *x = (key ? a.k + t * a.k_ld : a.q + t * a.q_ld) + h * hd;
                const bool rotate = o * 8 < nd;
                // the item's dims: d0.. and d1.. (four each)
                const int d0 = NEOX && rotate ? o * 4 : o * 8, d1 = NEOX && rotate ? nd / 2 + o * 4 : o * 8 + 4;
                uint32_t y[8];
                {
                    const float4 u = *reinterpret_cast<const float4 *>(x + d0), v = *reinterpret_cast<const float4 *>(x + d1);
                    const float w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                    cvt16_batch(C, w, y);
                }
                if (rotate) {
                    const uint4 cs = *reinterpret_cast<const uint4 *>(&s_cs[r * nd + o * 8]);   // of four pairs
                    const uint32_t z[4] = {cs.x, cs.y, cs.z, cs.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i0 = NEOX ? j : 2 * j, i1 = NEOX ? j + 4 : 2 * j + 1;
                        rotate_pair(s_g, y[i0], y[i1], z[j], y[i0], y[i1]);
                    }
                }
                if (!key) {
                    float *q = a.q_dst + t * a.q_dst_ld + h * hd;
                    *reinterpret_cast<float4 *>(q + d0) = make_float4(V(y[0]), V(y[1]), V(y[2]), V(y[3]));
                    *reinterpret_cast<float4 *>(q + d1) = make_float4(V(y[4]), V(y[5]), V(y[6]), V(y[7]));
                } else if (id >= 0) {
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = H(y[j]);
                    uint16_t *k = kv.k_pages + ((int64_t)id * n_head_kv + h) * head_codes + c * 8;
                    const uint2 lo = make_uint2(y[0] | y[1] << 16, y[2] | y[3] << 16);
                    const uint2 hi = make_uint2(y[4] | y[5] << 16, y[6] | y[7] << 16);
                    if (!NEOX) {
                        *reinterpret_cast<uint4 *>(k + (d0 >> 3) * page * 8) = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    } else {
                        *reinterpret_cast<uint2 *>(k + (d0 >> 3) * page * 8 + (d0 & 7)) = lo;
                        *reinterpret_cast<uint2 *>(k + (d1 >> 3) * page * 8 + (d1 & 7)) = hi;
                    }
                }
            } else if (id >= 0) {
                // four dims of the values, 64 / rows apart
                const int g = e - rot, f = (g & ~(span - 1)) * 4 + (g & (span - 1));
                const float *x = a.v + t * a.v_ld;
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = x[min(f + span * j, nk - 1)];
                int h = (int)((uint32_t)f / (uint32_t)hd), d = f - h * hd;
                uint16_t *v = kv.v_pages + (int64_t)id * n_head_kv * head_codes + (c >> 3) * hd * 8 + (c & 7);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (f + span * j < nk) v[h * head_codes + d * 8] = (uint16_t)C(__half2float(__float2half_rn(w[j])));
                    d += span;
                    while (d >= hd) d -= hd, h++;
                }
            }
        }
    }
}

// ---- attention --------------------------------------------------------------------

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // rows of any alignment

struct attn_paged_args {
    lnship_paged_kv kv;
    const float *q;
    float *dst;
    int64_t q_ld, dst_ld;
    float scale;          // times log2 e
    int window;           // 0: none
    int n_head, rep, page_sh, splits, tile_rows, min_per;
    bool vec;             // the queries' rows are 16-byte aligned
    // splits: sums [splits][ntok][n_head][head_dim], (maximum, total) [splits][ntok][n_head],
    // parts that a row has [ntok][n_head]
    float *sums;
    float2 *stats;
    int *used;
    // k_attn_decode's tiles [n_seq][pre_tiles][n_head_kv], and the flags of their groups of eight cells
    uint4 *pre;
    uint8_t *pre_ok;
    int pre_tiles;
};

constexpr int k_lo_sh = 11;             // the low halves are scaled by 2^11
constexpr float k_lo = 2048.0f, k_lo_inv = 1.0f / 2048.0f;
// the weights as halves are scaled by 2^k_p_sh; a running maximum may lag by
// k_p_lag binades, so they stay below the largest half
constexpr int k_p_sh = 10, k_p_lag = 5;

// x, y to a pair of halves, and what the rounding leaves, times 2^11, to
// another: together 22 bits of each, down to steps of 2^-35.  (The product of
// two low halves, 2^-22 of the whole, is left out.)
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const half2v h = {(_Float16)x, (_Float16)y};
    const half2v l = {(_Float16)((x - (float)h[0]) * k_lo), (_Float16)((y - (float)h[1]) * k_lo)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// (x k as a half, y k as a half) in a word, one rounding each
__device__ __forceinline__ uint32_t scaled_halves(float x, float y, float k) {
    uint32_t r;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,0,0]" : "=v"(r) : "v"(x), "s"(k));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel_hi:[0,0,0]" : "+v"(r) : "v"(y), "s"(k));
    return r;
}
// the halves of h times k, less x and y: (x - k h0, y - k h1) as halves
__device__ __forceinline__ uint32_t rest_halves(uint32_t h, float k, float x, float y) {
    uint32_t r;
    asm("v_fma_mixlo_f16 %0, %1, -%2, %3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "s"(k), "v"(x));
    asm("v_fma_mixhi_f16 %0, %1, -%2, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(r) : "v"(h), "s"(k), "v"(y));
    return r;
}

// Two xlns16 codes in a word to the split halves of their values.  The log
// field goes into the mantissa of 2^23 + log, one FMA makes it the exponent;
// 2^11 times the value stays within F32 and the split needs no other product.
// Log 0 (zero) becomes 2^-117, which rounds to zero in both halves.  Ten issue
// slots a code, four of them the power.
__device__ __forceinline__ void decode2(uint32_t w, uint32_t &hi, uint32_t &lo) {
    constexpr uint32_t magic = 0x4b000000u, top = 0x47ffu;   // 2^23; the largest log of a half
    typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
    const uint32_t l = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(
        __builtin_bit_cast(ushort2v, w & (k16_logmask << 16 | k16_logmask)), ushort2v{top, top}));
    constexpr float off = -(8388608.0f / 128 + 128 - k_lo_sh);
    const float x0 = __builtin_amdgcn_exp2f(
        fmaf(__uint_as_float(__builtin_amdgcn_perm(magic, l, 0x07060100u)), 1.0f / 128, off));
    const float x1 = __builtin_amdgcn_exp2f(
        fmaf(__uint_as_float(__builtin_amdgcn_perm(magic, l, 0x07060302u)), 1.0f / 128, off));
    const uint32_t h = scaled_halves(x0, x1, k_lo_inv), r = rest_halves(h, k_lo, x0, x1);
    const uint32_t sg = w & (k16_sign << 16 | k16_sign);
    hi = h ^ sg;
    lo = r ^ sg;
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

// Eight weights (scaled by 2^k_p_sh) to their halves, the rest of those, and
// the halves less the low halves' scale (for the values' low halves).  The
// rest is not scaled, so that all three products add up in one accumulator: a
// second one for the low ones takes 64 registers that 128 dims do not have.
// A half's steps end at 2^-24, so a weight is off by up to 2^-35 of its row's
// largest, and by as much again where its copy meets a value's low half.
// (k_p_sh 13 and k_p_lag 2 would make that an eighth, and rescale more often:
// 4096 tokens behind 4096 1076 us in place of 1066, a window of 1000 137 for 133.)
__device__ __forceinline__ void split_p(const float *p, frag &ph, frag &pl, frag &pc) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const half2v h = {(_Float16)p[j], (_Float16)p[j + 1]};
        const uint32_t hw = __builtin_bit_cast(uint32_t, h), r = rest_halves(hw, 1.0f, p[j], p[j + 1]);
        const half2v c = h * half2v{(_Float16)k_lo_inv, (_Float16)k_lo_inv};
        ph.u[j / 2] = hw;
        pl.u[j / 2] = r;
        pc.u[j / 2] = __builtin_bit_cast(uint32_t, c);
    }
}

__device__ __forceinline__ float4v mma(const frag &a, const frag &b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}
__device__ __forceinline__ float16v mma(const frag &a, const frag &b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}

// A tile of R rows of one sequence (row r: token r / rep, head r % rep of the
// kv head's group) and the cells that it sees.  Sequence s's tiles start at
// q_start[s] rep / R + s, which leaves each as many as it may need.
struct row_tile {
    int sq, t0, rows, r0;   // its sequence, that one's first token and rows, the tile's first row
    int pos0;               // position of token t0
    int c0, c1;             // cells [c0, c1) may be seen, c0 a multiple of 64
    int seen;               // the first cell that is (c1: none): pages before it may be any
    int blocks, per;        // blocks of 64 of them, and of a split
};
// r0 < 0: the tile has no rows.
__device__ __forceinline__ row_tile find_tile(const attn_paged_args &a, int tile, unsigned long long *err) {
    const lnship_paged_kv &kv = a.kv;
    const uint32_t R = (uint32_t)a.tile_rows, rep = (uint32_t)a.rep;
    auto first_tile = [&](int i) { return (int)((uint32_t)min(max(kv.q_start[i], 0), (int)kv.ntok) * rep / R) + i; };
    row_tile t;
    t.sq = wave_last_at_most((int)kv.n_seq, tile, first_tile);
    const int start = kv.q_start[t.sq], len = kv.kv_len[t.sq];   // (all loads before the first wait)
    const int64_t end = kv.q_start[t.sq + 1];
    t.t0 = min(max(start, 0), (int)kv.ntok);
    t.rows = (int)max(min(end, kv.ntok) - t.t0, (int64_t)0) * a.rep;
    t.r0 = (tile - first_tile(t.sq)) * a.tile_rows;
    if (t.r0 >= t.rows) t.r0 = -1;
    if (t.r0 < 0) return t;
    const int64_t pos0 = max((int64_t)len - end + t.t0, -((int64_t)1 << 30));
    const int last = (int)((uint32_t)(min(t.r0 + a.tile_rows, t.rows) - 1) / rep), first = (int)((uint32_t)t.r0 / rep);
    const int64_t cells = kv.table_ld << a.page_sh;
    if (err && pos0 + last >= cells && threadIdx.x == 0) index_fault(err, pos0 + last);
    t.pos0 = (int)min(pos0, ((int64_t)1 << 31) - 1 - t.rows);
    t.c1 = (int)max(min((int64_t)t.pos0 + last + 1, cells), (int64_t)0);
    t.seen = a.window > 0 ? max(0, min(t.pos0 + first - a.window + 1, t.c1)) : 0;
    t.c0 = t.seen & ~63;
    t.blocks = (t.c1 - t.c0 + 63) >> 6;
    t.per = max((t.blocks + a.splits - 1) / a.splits, a.min_per);
    return t;
}

// Where a row's sums go, and what they are multiplied by: divided into dst,
// or (splits) as they are into their part of the workspace, with the row's
// maximum and total (first: by the thread that writes those).
struct row_out {
    float *dst;
    float f;
};
__device__ __forceinline__ row_out out_row(const attn_paged_args &a, const row_tile &t, int split, int64_t tok, int head,
                                           float m, float l, bool first) {
    const int hd = (int)a.kv.head_dim;
    if (a.splits == 1) return {a.dst + tok * a.dst_ld + (int64_t)head * hd, m == -INFINITY ? 0.0f : 1.0f / l};
    const int64_t row = tok * a.n_head + head, part = split * a.kv.ntok * a.n_head + row;
    if (first) {
        a.stats[part] = make_float2(m, l);
        if (split == 0) a.used[row] = max((t.blocks + t.per - 1) / t.per, 1);
    }
    return {a.sums + part * hd, 1.0f};
}

// Eight queries of a row from dim d on.  Past head_dim other ones are loaded
// (in bounds) and made zeros: what is loaded is not written before it arrives,
// or every load would be waited for.
__device__ __forceinline__ void load_q(const float *q, int d, int hd, bool vec, float *x) {
    q += min(d, hd - 8);
    if (vec) {
        const float4 u = *reinterpret_cast<const float4 *>(q), v = *reinterpret_cast<const float4 *>(q + 4);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = q[j];
    }
}

// Few rows a sequence (single tokens): a wave takes 16 rows and, of their
// split's cells, every NW-th block of 32; the waves of a workgroup are joined at
// the end.  Scores are formed transposed, S^T = K Q^T, with the cells
// dealt to the rows of two 16 x 16 products so that a lane's eight scores are
// eight neighbouring cells of one row: as such they are the operand of
// O^T = V^T P^T, and both caches' layouts give a lane's share of K and V in
// 16-byte loads, straight from memory.  The next block's keys are loaded while
// this one's weights are formed, its values once this one's are decoded.
// Bound by HBM where the cache is long: 64 sequences of 100 to 8000 cells, 32 heads of
// 128 on 8, in 300 us, 3.7 TB/s of keys and values (a sum over memory reads 4.0); one of
// 131072 cells in 125 us, 4.2 TB/s.  300 cells of 9 heads of 64 on 3 take 9.4 us: the
// loads of lengths, pages, keys and values wait for each other.
template <int NB, bool FULL, int NW>   // 32-wide groups of head_dim; whether it fills them; waves
__global__ __launch_bounds__(NW * 64, NW == 8 ? 2 : NB <= 4 ? 3 : 1) void k_attn_paged(attn_paged_args a, unsigned long long *err) {
    const lnship_paged_kv &kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int rep = a.rep, kvh = blockIdx.y, split = blockIdx.z, hd = (int)kv.head_dim, page = (int)kv.page;
    constexpr int step = NW * 32;
    constexpr int slots = NB <= 2 ? NW : NB <= 4 ? 4 : 2;   // waves that put their sums into LDS at once
    __shared__ float s_m[NW][16], s_l[NW][16], s_qs[16];
    __shared__ float s_o[slots][16][NB * 32 + 1];
    __shared__ uint4 s_q[2][NB][64];   // the queries' split halves, as the products' operands

    const row_tile T = find_tile(a, blockIdx.x, err);
    if (T.r0 < 0 || (split > 0 && split * T.per >= T.blocks)) return;
    const int cend = min(T.c1, T.c0 + (split + 1) * T.per * 64);

    // the lane's row
    const bool have = T.r0 + n < T.rows;
    const int row = have ? T.r0 + n : T.r0, tok = T.t0 + (int)((uint32_t)row / (uint32_t)rep);
    const int head = kvh * rep + (int)((uint32_t)row % (uint32_t)rep);
    const int pos = min(T.pos0 + tok - T.t0, T.c1 - 1);
    const int lo_cell = a.window > 0 ? T.pos0 + tok - T.t0 - a.window : -1;   // cells at and below are hidden

    const int32_t *table = kv.table + (int64_t)T.sq * kv.table_ld;
    const int64_t head_codes = (int64_t)page * hd, page_codes = kv.n_head_kv * head_codes;
    const uint16_t *kbase = kv.k_pages + kvh * head_codes, *vbase = kv.v_pages + kvh * head_codes;
    // the lane's cells of a block: as a row of the key products (4 of each of
    // the two), and of its eight scores
    const int kcell = 8 * (n >> 2), vcell = 8 * g;
    // the page of cell c (of hidden cells: another's, whatever it holds is finite)
    auto page_of = [&](int c) { return table[min(c, cend - 1) >> a.page_sh]; };
    auto sound = [&](int id) { return (uint32_t)id < (uint32_t)kv.n_pages; };
    // (past head_dim the last dims are loaded again: the queries are zeros there,
    // and those sums are not written)
    uint4 kc[2][NB], vc[2 * NB];
    auto load_k = [&](int cb, int id) {
        const int c = (cb + kcell) & (page - 1);
        const uint16_t *k = kbase + (sound(id) ? id : 0) * page_codes + (c + (n & 3)) * 8;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int d8 = FULL ? i * 4 + g : min(i * 4 + g, hd / 8 - 1);
                kc[t][i] = *reinterpret_cast<const uint4 *>(k + (d8 * page + 4 * t) * 8);
            }
    };
    auto load_v = [&](int cb, int id) {
        const uint16_t *v = vbase + (sound(id) ? id : 0) * page_codes + ((cb + vcell) & (page - 1)) * hd;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            const int d = FULL ? i * 16 + n : min(i * 16 + n, hd - 1);
            vc[i] = *reinterpret_cast<const uint4 *>(v + d * 8);
        }
    };

    float4v o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) o[i] = float4v{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    int cb = T.c0 + split * T.per * 64 + wave * 32;
    // (a page's number is used before the next one is loaded into its place, so
    // that no copy of it waits for loads behind it)
    int vid = 0, kid = 0;
    bool vok = false;
    auto sound_v = [&](int cb) {
        vok = cb + vcell < cend && sound(vid);
        if (cb + vcell < cend && !vok) {
            asm volatile("");   // (few blocks need the rest)
            if (cb + vcell + 7 >= T.seen) index_fault(err, vid);
        }
    };
    if (cb < cend) {
        kid = page_of(cb + kcell);
        vid = page_of(cb + vcell);
        load_k(cb, kid);
        kid = page_of(cb + step + kcell);
        sound_v(cb);
        load_v(cb, vid);
        vid = page_of(cb + step + vcell);
    }
    // the queries as halves, scaled by the row's largest to at most 2: by the
    // first wave, for all
    if (wave == 0) {
        float x[NB][8], mx = 0.0f;
        const float *q = a.q + tok * a.q_ld + (int64_t)head * hd;
#pragma unroll
        for (int b = 0; b < NB; b++) load_q(q, b * 32 + g * 8, FULL ? NB * 32 : hd, a.vec, x[b]);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!FULL && b * 32 + g * 8 >= hd) x[b][j] = 0.0f;
                mx = fmaxf(mx, fabsf(x[b][j]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int e = (int)(f32_bits(mx) >> 23) - 127;   // -127 for zeros
#pragma unroll
        for (int b = 0; b < NB; b++) {
            frag hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j += 2) split2(ldexpf(x[b][j], -e), ldexpf(x[b][j + 1], -e), hi.u[j / 2], lo.u[j / 2]);
            s_q[0][b][lane] = hi.w;
            s_q[1][b][lane] = lo.w;
        }
        if (g == 0) s_qs[n] = ldexpf(a.scale, e);
    }
    __syncthreads();
    const float qs = s_qs[n];
    for (; cb < cend; cb += step) {
        float4v sh[2], sx[2];
        sh[0] = sh[1] = sx[0] = sx[1] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NB; i++) {
            frag qh, ql;
            qh.w = s_q[0][i][lane];
            ql.w = s_q[1][i][lane];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                frag kh, kl;
                decode8(kc[t][i], kh, kl);
                sh[t] = mma(kh, qh, sh[t]);
                sx[t] = mma(kl, qh, sx[t]);
                sx[t] = mma(kh, ql, sx[t]);
            }
        }
        load_k(cb + step, kid);
        kid = page_of(cb + 2 * step + kcell);
        float s[8], mb = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int cell = cb + vcell + j;
            s[j] = (sh[j >> 2][j & 3] + k_lo_inv * sx[j >> 2][j & 3]) * qs;
            if (!vok || cell > pos || cell <= lo_cell) s[j] = -INFINITY;
            mb = fmaxf(mb, s[j]);
        }
        if (__any(mb > m + k_p_lag)) {   // the first block, and where the maximum has grown far
            mb = fmaxf(mb, __shfl_xor(mb, 16));
            mb = fmaxf(mb, __shfl_xor(mb, 32));
            const float mn = fmaxf(m, mb);
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) o[i] *= alpha;
        }
        const float ms = (m == -INFINITY ? 0.0f : m) - k_p_sh;
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(s[j] - ms);
            l += p[j];
        }
        frag ph, pl, pc;
        split_p(p, ph, pl, pc);
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            frag vh, vl;
            decode8(vc[i], vh, vl);
            o[i] = mma(vh, ph, o[i]);
            o[i] = mma(vh, pl, o[i]);
            o[i] = mma(vl, pc, o[i]);
        }
        sound_v(cb + step);
        load_v(cb + step, vid);
        vid = page_of(cb + 2 * step + vcell);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' parts joined, in the waves' order
    if (g == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    __syncthreads();
    float M = s_m[0][n];
#pragma unroll
    for (int w = 1; w < NW; w++) M = fmaxf(M, s_m[w][n]);
    const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    for (int w = 0; w < NW; w += slots) {
        if (wave >= w && wave < w + slots) {
#pragma unroll
            for (int i = 0; i < 2 * NB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float &x = s_o[wave - w][n][i * 16 + g * 4 + j];
                    x = (w ? x : 0.0f) + o[i][j] * f;
                }
        }
        __syncthreads();
    }
    // a row's elements, on as many threads as there are for a row
    constexpr int of = NW * 4;
    const int rr = threadIdx.x / of, row2 = T.r0 + rr;
    if (row2 >= T.rows) return;
    const int tok2 = T.t0 + (int)((uint32_t)row2 / (uint32_t)rep), head2 = kvh * rep + (int)((uint32_t)row2 % (uint32_t)rep);
    float M2 = -INFINITY, L2 = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) M2 = fmaxf(M2, s_m[w][rr]);
    if (M2 != -INFINITY)
#pragma unroll
        for (int w = 0; w < NW; w++) L2 += s_l[w][rr] * __builtin_amdgcn_exp2f(s_m[w][rr] - M2);
    const row_out out = out_row(a, T, split, tok2, head2, M2, L2, threadIdx.x % of == 0);
    for (int d = threadIdx.x % of; d < hd; d += of) {
        float x = s_o[0][rr][d];
#pragma unroll
        for (int w = 1; w < slots; w++) x += s_o[w][rr][d];
        out.dst[d] = x * out.f;
    }
}

// A barrier that waits for LDS alone: loads from memory stay in flight; and one
// that waits for them too (copies into LDS among them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ void copy_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Copies 16 bytes a lane from memory to LDS, from `to` on in the lanes' order,
// without a register between.
__device__ __forceinline__ void copy_to_lds(const uint4 *from, uint4 *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// 64 cells of one kv head as split halves, in the order in which the products of
// chunk_rows read them (a lane's 16 bytes of an operand behind the lane
// before's): for each block of 32 cells B units of the keys' high halves, of
// their low ones, of the values' high and low ones.  Past head_dim the last dims
// are repeated: the queries are zeros there, and those sums are not written.
template <int NB>
struct tile_of {
    static constexpr int HD = NB * 32;
    static constexpr int B = 32 * HD / 8;   // 16-byte units of 32 cells' keys, and values
    static constexpr int U = 2 * B;
};

// A workgroup of NT threads that makes such tiles of the cells [.., cend) of one
// sequence, of which those before `seen` are seen by no row: a thread loads its units' codes ahead, then decodes them.  Unit u of
// the keys: dims u / C * 8.., cell u % C of the tile's C (the same for all of a
// thread's); of the values: cells u / HD * 8.., dim u % HD.
template <int NB, int NT, int C = 64>
struct tile_maker {
    static constexpr int HD = tile_of<NB>::HD, B = tile_of<NB>::B, U = C / 32 * B, UT = (U + NT - 1) / NT;
    const int32_t *table;
    const uint16_t *kbase, *vbase;
    int64_t page_codes;
    int seen, cend, page_sh, page, hd, n_pages, tid;
    unsigned long long *err;
    uint4 kc[UT], vc[UT];
    int kid, vid[UT];   // the pages of the next units to load

    __device__ __forceinline__ tile_maker(const lnship_paged_kv &kv, int sq, int kvh, int sh, int first_seen, int end, int thread,
                                          unsigned long long *e)
        : table(kv.table + (int64_t)sq * kv.table_ld), seen(first_seen), cend(end), page_sh(sh), page((int)kv.page), hd((int)kv.head_dim),
          n_pages((int)kv.n_pages), tid(thread), err(e) {
        const int64_t head_codes = (int64_t)page * hd;
        page_codes = kv.n_head_kv * head_codes;
        kbase = kv.k_pages + kvh * head_codes;
        vbase = kv.v_pages + kvh * head_codes;
    }
    __device__ __forceinline__ bool has(int i) const { return (i + 1) * NT <= U || tid + i * NT < U; }
    // the page of cell c (of hidden cells: another's, whatever it holds is finite)
    __device__ __forceinline__ int page_of(int c) const { return table[min(c, cend - 1) >> page_sh]; }
    __device__ __forceinline__ bool sound(int id) const { return (uint32_t)id < (uint32_t)n_pages; }
    __device__ __forceinline__ void pages(int cb) {
        kid = page_of(cb + (tid & (C - 1)));
#pragma unroll
        for (int i = 0; i < UT; i++) vid[i] = page_of(cb + (tid + i * NT) / HD * 8);
    }
    __device__ __forceinline__ void load(int cb) {
        const uint16_t *k = kbase + (sound(kid) ? kid : 0) * page_codes + ((cb + (tid & (C - 1))) & (page - 1)) * 8;
#pragma unroll
        for (int i = 0; i < UT; i++) {
            const int d8 = (tid + i * NT) / C;
            kc[i] = *reinterpret_cast<const uint4 *>(k + min(d8, hd / 8 - 1) * page * 8);
        }
#pragma unroll
        for (int i = 0; i < UT; i++) {
            const int c8 = (tid + i * NT) / HD, d = (tid + i * NT) % HD;
            const uint16_t *v = vbase + (sound(vid[i]) ? vid[i] : 0) * page_codes + ((cb + c8 * 8) & (page - 1)) * hd;
            vc[i] = *reinterpret_cast<const uint4 *>(v + min(d, hd - 1) * 8);
        }
    }
    // Whether the pages of the thread's values, for the tile at cb, are sound.
    // Taken from the pages' numbers before the next ones are loaded, so that no
    // copy of a number waits for its load (and with it for all before it).
    __device__ __forceinline__ uint32_t sound_pages(int cb) const {
        uint32_t ok = 0;
#pragma unroll
        for (int i = 0; i < UT; i++) {
            const int c = cb + (tid + i * NT) / HD * 8;
            const bool in = has(i) && c < cend;
            if (in && sound(vid[i])) ok |= 1u << i;
            else if (in) {
                asm volatile("");   // (few tiles need the rest)
                if (c + 7 >= seen) index_fault(err, vid[i]);
            }
        }
        return ok;
    }
    // decodes the loaded codes into the tile s; its groups of eight cells' flags into oks
    __device__ __forceinline__ void store(uint4 *s, uint32_t ok, uint8_t *oks) const {
        // the cell's row of its block's key product: a lane's 16 results are
        // then cells 8 h + 0..7 and 16 + 8 h + 0..7 of the block
        const int cell = tid & (C - 1), in = cell & 31;
        const int row = 8 * ((in >> 4) * 2 + ((in >> 2) & 1)) + 4 * ((in >> 3) & 1) + (in & 3);
#pragma unroll
        for (int i = 0; i < UT; i++) {
            frag hi, lo;
            decode8(kc[i], hi, lo);
            if (!has(i)) continue;
            const int d8 = (tid + i * NT) / C;
            uint4 *to = s + (cell >> 5) * 4 * B + (d8 >> 1) * 64 + (d8 & 1) * 32 + row;
            to[0] = hi.w;
            to[B] = lo.w;
        }
#pragma unroll
        for (int i = 0; i < UT; i++) {
            frag hi, lo;
            decode8(vc[i], hi, lo);
            if (!has(i)) continue;
            const int c8 = (tid + i * NT) / HD, d = (tid + i * NT) % HD;
            uint4 *to = s + (c8 >> 2) * 4 * B + (d >> 5) * 128 + ((c8 >> 1) & 1) * 64 + (c8 & 1) * 32 + (d & 31);
            to[2 * B] = hi.w;
            to[3 * B] = lo.w;
            if (oks && d == 0) oks[c8] = ok >> i & 1;
        }
    }
    // The same for the tiles [cb, cend), one behind the other: loads the first and
    // decodes it, then each next one, its loads ahead of the one before's decoding.
    uint32_t ok_next;
    __device__ __forceinline__ void first(int cb, uint4 *s, uint8_t *oks) {
        if (cb >= cend) return;
        pages(cb);
        load(cb);
        ok_next = sound_pages(cb);
        pages(cb + C);
        next(cb, s, oks);
    }
    __device__ __forceinline__ void next(int cb, uint4 *s, uint8_t *oks) {
        if (cb >= cend) return;
        store(s, ok_next, oks);
        load(cb + C);   // (past the last tile: other cells of a page, not used)
        ok_next = sound_pages(cb + C);
        pages(cb + 2 * C);
    }
};

// The cells that chunks see, decoded into the workspace, for k_attn_tiles to
// copy: a workgroup takes every gridDim.x-th tile of a sequence and kv head.
// Eight bytes are written for two: 8192 cells of 8 heads of 128 take 18 us.
template <int NB>
__global__ __launch_bounds__(256) void k_attn_decode(attn_paged_args a, unsigned long long *err) {
    const lnship_paged_kv &kv = a.kv;
    const int nkv = (int)kv.n_head_kv, kvh = (int)(blockIdx.y % (uint32_t)nkv);
    for (int sq = (int)(blockIdx.y / (uint32_t)nkv); sq < (int)kv.n_seq; sq += (int)(gridDim.y / (uint32_t)nkv)) {
        const int64_t start = kv.q_start[sq], end = kv.q_start[sq + 1];
        const int cend = (int)max(min((int64_t)kv.kv_len[sq], kv.table_ld << a.page_sh), (int64_t)0);
        if (end <= start) continue;
        // the first cell that the sequence's first token sees
        const int64_t first = kv.kv_len[sq] - (end - start) - a.window + 1;
        const int seen = a.window > 0 ? (int)min(max(first, (int64_t)0), (int64_t)cend) : 0;
        tile_maker<NB, 256> t(kv, sq, kvh, a.page_sh, seen, cend, threadIdx.x, err);
        for (int i = (seen >> 6) + (int)blockIdx.x; i * 64 < cend; i += (int)gridDim.x) {
            t.pages(i * 64);
            t.load(i * 64);
            const uint32_t ok = t.sound_pages(i * 64);
            const int64_t at = (int64_t)sq * a.pre_tiles + i;
            t.store(a.pre + (at * nkv + kvh) * 4 * tile_of<NB>::U, ok, kvh == 0 ? a.pre_ok + at * 8 : nullptr);
        }
    }
}

// A wave's 32 rows of a tile and their running sums.  Products are 32 x 32 x 16,
// transposed as above; a lane has 16 scores of one row (row n, with the lane 32
// on, which has the block's other cells).
template <int NB>
struct chunk_rows {
    static constexpr int KK = NB * 2, B = tile_of<NB>::B;
    int h, tok, head, pos, lo_cell;
    int wfirst, wlast, all_lo, any_lo;   // what all of the wave's rows see, and any does
    bool have, any;
    frag qh[KK], ql[KK];
    float qs, m, l;
    float16v o[NB];

    __device__ __forceinline__ void place(const attn_paged_args &a, const row_tile &T, int kvh, int wrow) {
        const int lane = threadIdx.x & 63, n = lane & 31;
        const uint32_t rep = (uint32_t)a.rep;
        h = lane >> 5;
        any = wrow < T.rows;
        have = wrow + n < T.rows;
        const int row = have ? wrow + n : min(wrow, T.rows - 1);
        tok = T.t0 + (int)((uint32_t)row / rep);
        head = kvh * a.rep + (int)((uint32_t)row % rep);
        pos = min(T.pos0 + tok - T.t0, T.c1 - 1);
        lo_cell = a.window > 0 ? T.pos0 + tok - T.t0 - a.window : -1;
        wfirst = T.pos0 + (int)((uint32_t)min(wrow, T.rows - 1) / rep);
        wlast = T.pos0 + (int)((uint32_t)(min(wrow + 32, T.rows) - 1) / rep);
        all_lo = a.window > 0 ? wlast - a.window : -1;
        any_lo = a.window > 0 ? wfirst - a.window : -1;
    }
    // the queries as halves, scaled by the row's largest to at most 2
    __device__ __forceinline__ void load(const attn_paged_args &a) {
        const int hd = (int)a.kv.head_dim;
        float x[KK][8], mx = 0.0f;
        const float *q = a.q + tok * a.q_ld + (int64_t)head * hd;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) load_q(q, kk * 16 + h * 8, hd, a.vec, x[kk]);
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (kk * 16 + h * 8 >= hd) x[kk][j] = 0.0f;
                mx = fmaxf(mx, fabsf(x[kk][j]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int e = (int)(f32_bits(mx) >> 23) - 127;   // -127 for zeros
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                split2(ldexpf(x[kk][j], -e), ldexpf(x[kk][j + 1], -e), qh[kk].u[j / 2], ql[kk].u[j / 2]);
        qs = ldexpf(a.scale, e);
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; i++) o[i] = float16v{};
    }
    // the block of 32 cells from b0 on, at s in LDS; ok: a byte for each eight of
    // them, 1 where they lie in a page; c1: the end of the tile's cells
    __device__ __forceinline__ void block(const uint4 *tile, int b0, uint32_t ok, int c1) {
        if (!any || b0 > wlast || b0 + 31 <= any_lo) return;
        const frag *s = reinterpret_cast<const frag *>(tile) + (threadIdx.x & 63);
        float16v sh{}, sx{};
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            const frag kh = s[kk * 64], kl = s[B + kk * 64];
            sh = mma(kh, qh[kk], sh);
            sx = mma(kl, qh[kk], sx);
            sx = mma(kh, ql[kk], sx);
        }
        float p[16], mb = -INFINITY;
        const float sub = (m == -INFINITY ? 0.0f : m) - k_p_sh;
#pragma unroll
        for (int j = 0; j < 16; j++) p[j] = fmaf(sx[j], qs * k_lo_inv, fmaf(sh[j], qs, -sub));
        if (b0 + 31 > wfirst || b0 + 31 >= c1 || b0 <= all_lo || ok != 0x01010101u) {
            asm volatile("");   // a branch: few blocks need it
            const bool ok0 = ok >> (8 * h) & 1, ok1 = ok >> (16 + 8 * h) & 1;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int cell = b0 + (j >> 3) * 16 + h * 8 + (j & 7);
                if (!(j < 8 ? ok0 : ok1) || cell > pos || cell <= lo_cell) p[j] = -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 16; j++) mb = fmaxf(mb, p[j]);
        // p holds the scores less sub: the first block, and where the maximum has grown far
        if (__any(m == -INFINITY ? mb != -INFINITY : mb > (float)(k_p_sh + k_p_lag))) {
            mb = fmaxf(mb, __shfl_xor(mb, 32));
            const float mn = fmaxf(m, mb + sub);
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float more_sub = (mn == -INFINITY ? 0.0f : mn) - k_p_sh - sub;
#pragma unroll
            for (int j = 0; j < 16; j++) p[j] -= more_sub;
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; i++) o[i] *= alpha;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
            p[j] = __builtin_amdgcn_exp2f(p[j]);
            l += p[j];
        }
        frag ph[2], pl[2], pc[2];
        split_p(p, ph[0], pl[0], pc[0]);
        split_p(p + 8, ph[1], pl[1], pc[1]);
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const frag vh = s[2 * B + i * 128 + t * 64], vl = s[3 * B + i * 128 + t * 64];
                o[i] = mma(vh, ph[t], o[i]);
                o[i] = mma(vh, pl[t], o[i]);
                o[i] = mma(vl, pc[t], o[i]);
            }
    }
    __device__ __forceinline__ void write(const attn_paged_args &a, const row_tile &T, int split) {
        const int hd = (int)a.kv.head_dim;
        l += __shfl_xor(l, 32);
        if (!have) return;
        const row_out out = out_row(a, T, split, tok, head, m, l, h == 0);
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int d = i * 32 + 2 * j + 4 * h;
                const float4v x = {o[i][j] * out.f, o[i][j + 1] * out.f, o[i][j + 2] * out.f, o[i][j + 3] * out.f};
                if (d < hd) *reinterpret_cast<float4u *>(out.dst + d) = x;
            }
    }
};

// the tile, kv head and split of a workgroup: kv heads side by side (on the
// XCDs' L2s), the last tiles (most cells) first
__device__ __forceinline__ int chunk_tile(int nkv, int &kvh) {
    kvh = (int)(blockIdx.x % (uint32_t)nkv);
    return (int)(gridDim.x / (uint32_t)nkv) - 1 - (int)(blockIdx.x / (uint32_t)nkv);
}

// Many rows a sequence (prompts, chunks), over cells that k_attn_decode has
// decoded: NW waves of 32 rows go over them 32 at a time, from two LDS buffers;
// while one is multiplied the next block is copied into the other, without
// registers.  Two or more workgroups to a CU, where registers leave room: a
// barrier holds one of them up, and the other's waves multiply meanwhile.
// Bound by the matrix cores: 4096 tokens behind 4096 cells, 32 heads of 128 on 8, in
// 1043 to 1090 us (box to box), of which k_attn_decode takes 18: 1140 TFLOP/s in
// f16, three products for one, where a library's large product reaches 1163; the
// clock falls from 2.15 to 1.76 GHz under this load.  Two prompts of 1900 to 2500
// tokens, 32 heads of 64 on 8, in a window of 1000: 134 us.
template <int NB, int NW>
__global__ __launch_bounds__(NW * 64, NB <= 2 ? 3 : 2) void k_attn_tiles(attn_paged_args a, unsigned long long *err) {
    constexpr int B = tile_of<NB>::B, NT = NW * 64;
    static_assert(4 * B % NT == 0, "whole copies");
    __shared__ uint4 s_tile[2][4 * B];
    const int tid = threadIdx.x, wave = tid >> 6, nkv = (int)a.kv.n_head_kv, split = blockIdx.y;
    int kvh;
    const int tile = chunk_tile(nkv, kvh);
    const row_tile T = find_tile(a, tile, err);
    if (T.r0 < 0 || (split > 0 && split * T.per >= T.blocks)) return;
    const int cbeg = T.c0 + split * T.per * 64, cend = min(T.c1, cbeg + T.per * 64);
    const uint4 *from = a.pre + ((int64_t)T.sq * a.pre_tiles * nkv + kvh) * 8 * B + tid;
    const uint32_t *oks = reinterpret_cast<const uint32_t *>(a.pre_ok) + (int64_t)T.sq * a.pre_tiles * 2;
    uint32_t ok_next = 0;
    auto copy = [&](int b0, int buf) {
        const uint4 *f = from + (int64_t)(b0 >> 6) * nkv * 8 * B + (b0 >> 5 & 1) * 4 * B;
#pragma unroll
        for (int i = 0; i < 4 * B / NT; i++) copy_to_lds(f + i * NT, &s_tile[buf][i * NT + wave * 64]);
        ok_next = oks[b0 >> 5];
    };
    if (cbeg < cend) copy(cbeg, 0);
    chunk_rows<NB> r;
    r.place(a, T, kvh, T.r0 + wave * 32);
    r.load(a);
    copy_barrier();
    int buf = 0;
    for (int b0 = cbeg; b0 < cend; b0 += 32, buf ^= 1) {
        const uint32_t ok = ok_next;
        if (b0 + 32 < cend) copy(b0 + 32, buf ^ 1);
        r.block(s_tile[buf], b0, ok, T.c1);
        copy_barrier();
    }
    r.write(a, T, split);
}

// The same where a cell meets one tile or two of a sequence, or the tables' cells
// are more than the workspace holds decoded: NW waves go over C cells at a time
// and decode the codes themselves, each once a workgroup, by the thread that loaded
// it a tile before, into the other of two LDS buffers.  Bound by the decoding and
// the products in turn, and with few workgroups by the slowest: 9 conversations of 5
// to 301 tokens behind up to 1777, 9 heads of 64 on 3, in 34 us with the join.
template <int NB, int NW, int C>   // 32-wide groups of head_dim; waves; cells of a tile
__global__ __launch_bounds__(NW * 64, NW == 4 ? 2 : 1) void k_attn_chunk(attn_paged_args a, unsigned long long *err) {
    constexpr int B = tile_of<NB>::B, buf_units = C / 32 * 4 * B;
    extern __shared__ uint4 s_cells[];         // [2][buf_units]
    __shared__ alignas(16) uint8_t s_ok[2][C / 8];   // whether a tile's groups of eight cells lie in a page
    const int wave = threadIdx.x >> 6, split = blockIdx.y;
    int kvh;
    const int tile = chunk_tile((int)a.kv.n_head_kv, kvh);
    const row_tile T = find_tile(a, tile, err);
    if (T.r0 < 0 || (split > 0 && split * T.per >= T.blocks)) return;
    const int cbeg = T.c0 + split * T.per * 64, cend = min(T.c1, cbeg + T.per * 64);
    const int tid = threadIdx.x;
    auto cells = [&](int buf) { return s_cells + buf * buf_units; };
    chunk_rows<NB> r;
    auto blocks = [&](int cb, int buf) {
#pragma unroll 1
        for (int blk = 0; blk < C / 32; blk++) {
            const uint32_t ok = (uint32_t)__builtin_amdgcn_readfirstlane(
                (int)*reinterpret_cast<const uint32_t *>(&s_ok[buf][blk * 4]));
            r.block(cells(buf) + blk * 4 * B, cb + blk * 32, ok, T.c1);
        }
    };
    if (NW == 8 && T.rows - T.r0 <= NW * 16) {
        // Rows for half of the waves: the others decode meanwhile.  (33 sequences of 6
        // to 27 tokens behind 640 to 5125 cells, 32 heads of 128 on 8: 244 to 259 us, all
        // waves decoding 283 to 296.)
        if (wave >= NW / 2) {
            tile_maker<NB, NW * 32, C> maker(a.kv, T.sq, kvh, a.page_sh, T.seen, cend, tid - NW * 32, err);
            maker.first(cbeg, cells(0), s_ok[0]);
            lds_barrier();
            int buf = 0;
            for (int cb = cbeg; cb < cend; cb += C, buf ^= 1) {
                maker.next(cb + C, cells(buf ^ 1), s_ok[buf ^ 1]);
                lds_barrier();
            }
            return;
        }
        r.place(a, T, kvh, T.r0 + wave * 32);
        r.load(a);
        lds_barrier();
        int buf = 0;
        for (int cb = cbeg; cb < cend; cb += C, buf ^= 1) {
            blocks(cb, buf);
            lds_barrier();
        }
        r.write(a, T, split);
        return;
    }
    tile_maker<NB, NW * 64, C> maker(a.kv, T.sq, kvh, a.page_sh, T.seen, cend, tid, err);
    maker.first(cbeg, cells(0), s_ok[0]);
    r.place(a, T, kvh, T.r0 + wave * 32);
    r.load(a);
    lds_barrier();
    int buf = 0;
    for (int cb = cbeg; cb < cend; cb += C, buf ^= 1) {
        blocks(cb, buf);
        maker.next(cb + C, cells(buf ^ 1), s_ok[buf ^ 1]);
        lds_barrier();
    }
    r.write(a, T, split);
}

// The splits' parts of a row joined, in a fixed order, by one wave (four rows a
// workgroup) or, many parts, by the workgroup's four: head_dim / 4 lanes read a
// part, the others other parts beside it.  Bound by the launch and one read of the
// parts: 6.6 us for the rows of 9 conversations, 9 heads of 64.
template <int W>   // waves of a row
__global__ __launch_bounds__(256) void k_attn_paged_join(attn_paged_args a) {
    constexpr int S = W == 4 ? 256 : 64;   // parts at most
    __shared__ float s_f[4 / W][S], s_red[2][4];
    __shared__ float4 s_o[4][64];
    const int hd = (int)a.kv.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t rows = a.kv.ntok * a.n_head;
    const int64_t row = W == 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    const int64_t tok = row / a.n_head;
    const int at = W == 4 ? tid : lane;
    // (what no part has written is loaded too, beside what says so, and not used;
    // an unsound q_start may leave rows out)
    const int64_t own = min(row, rows - 1);
    const float2 part = a.stats[min(at, a.splits - 1) * rows + own];
    const int parts = a.used[own];
    const bool in = row < rows && tok >= a.kv.q_start[0] && tok < a.kv.q_start[a.kv.n_seq];
    if (W == 4 && !in) return;
    const int used = in ? max(1, min(parts, a.splits)) : 0;
    const float2 st = at < used ? part : make_float2(-INFINITY, 0.0f);
    auto reduce = [&](float v, bool sum) {
        for (int d = 32; d; d >>= 1) {
            const float y = __shfl_xor(v, d);
            v = sum ? v + y : fmaxf(v, y);
        }
        if (W == 1) return v;
        float *r = s_red[sum];
        if (lane == 0) r[wave] = v;
        __syncthreads();
        return sum ? r[0] + r[1] + r[2] + r[3] : fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
    };
    const float M = reduce(st.x, false);
    const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.x - M);
    float *sf = s_f[W == 4 ? 0 : wave];
    if (at < S) sf[at] = f;
    const float L = reduce(st.y * f, true);
    __syncthreads();
    const int lanes = hd >> 2, par = 64 / lanes, sub = lane / lanes, d4 = lane - sub * lanes;
    float4 s = make_float4(0, 0, 0, 0);
    if (sub < par) {
        const int64_t step = rows * hd;
        const float4 *w = reinterpret_cast<const float4 *>(a.sums + row * hd) + d4;
        const int inc = par * W;
#pragma unroll 8
        for (int i = (W == 4 ? wave * par : 0) + sub; i < used; i += inc) {
            const float4 v = w[i * (step >> 2)];
            const float fi = sf[i];
            s.x = fmaf(v.x, fi, s.x), s.y = fmaf(v.y, fi, s.y), s.z = fmaf(v.z, fi, s.z), s.w = fmaf(v.w, fi, s.w);
        }
    }
    s_o[wave][lane] = s;
    __syncthreads();
    if (!in || (W == 4 && wave > 0) || lane >= lanes) return;
    const float inv = M == -INFINITY ? 0.0f : 1.0f / L;
    float4 t = make_float4(0, 0, 0, 0);
    for (int w = W == 4 ? 0 : wave; w <= (W == 4 ? 3 : wave); w++)
        for (int q = 0; q < par; q++) {
            const float4 v = s_o[w][q * lanes + lane];
            t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
        }
    float *dst = a.dst + tok * a.dst_ld + (row - tok * a.n_head) * hd + lane * 4;
    dst[0] = t.x * inv, dst[1] = t.y * inv, dst[2] = t.z * inv, dst[3] = t.w * inv;
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
    if (kv->ntok > 0xfffff0 || kv->n_seq > 0x7fffff || kv->n_head_kv > 65535 || kv->n_pages > 0x7fffffff ||
        kv->table_ld > 0x3fffffff / kv->page)
        return fail(LNSHIP_ERANGE, "paged cache: too large%s");
    if (ptrs && kv->ntok && kv->n_seq) {
        if (!kv->k_pages || !kv->v_pages || !kv->q_start || !kv->kv_len || (!kv->table && kv->table_ld))
            return fail(LNSHIP_EINVAL, "paged cache: null pointer%s");
        if (((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15)
            return fail(LNSHIP_EINVAL, "paged cache: pages not 16-byte aligned%s");
    }
    return 0;
}

// Whether out's rows (n of w floats, out_ld apart) are x's, or share no memory with
// them: of rows equally far apart, one may lie in the gaps of the other.
static bool same_or_apart(const float *x, int64_t x_ld, const float *out, int64_t out_ld, int64_t w, int64_t n) {
    if (x == out && (x_ld == out_ld || n == 1)) return true;
    const int64_t a = (int64_t)(uintptr_t)x, b = (int64_t)(uintptr_t)out, bytes = w * 4;
    if (a + (n - 1) * x_ld * 4 + bytes <= b || b + (n - 1) * out_ld * 4 + bytes <= a) return true;
    if (x_ld != out_ld) return false;
    const int64_t step = x_ld * 4, d = ((b - a) % step + step) % step;
    return d >= bytes && step - d >= bytes;
}

static int log2_of(int64_t page) {
    int sh = 0;
    while ((int64_t)1 << sh < page) sh++;
    return sh;
}

// How a call runs: k_attn_tiles (pre) or k_attn_chunk with `waves` waves, or (0) k_attn_paged; rows
// of a tile, tiles, and the parts that a row's cells are split into.
struct attn_plan {
    int waves, tile_rows, splits, min_per;
    bool pre;   // cells decoded once, into the workspace
    int64_t tiles;
    // the workspace: bytes of the splits' parts, of the decoded tiles, of their flags
    int64_t parts_bytes, pre_bytes, ok_bytes, pre_tiles;
};
// The rules go by what the host knows, the rows of all sequences and the tables'
// cells, so that a captured graph runs the same kernels whatever its lengths.  They
// were measured on batches of sequences that are alike, behind tables as wide as the
// longest.  What they cost elsewhere: one kernel serves single tokens and a chunk in
// one call (32 heads of 128 on 8, 64 tokens over 4000 cells and a chunk behind 4000: of
// 512 tokens 579 us, apart 232 and 146; of 4096 1675, apart 230 and 1021), and a wide
// table stands for long caches (one token over 300 cells, 9 heads of 64 on 3, behind a
// table of 131072 14.4 us, of 304 9.2).
//
// Few rows a sequence, or little work: k_attn_paged, whose tiles are 16 rows and
// whose loads go straight to registers.  Otherwise the chunks' kernels, which
// read a cell once for 128 or 256 rows but take longer to start.  Measured with
// 16-row tiles and chunks (us): 8 sequences of 8 tokens over 500 cells, 32 heads
// of 128 on 8: 20.0 and 24.3; of 32 tokens (2^29 below): 45.5 and 31.5; 32 of 16 over
// 1000: 126 and 81; 9 heads of 64 on 3, 8 of 64 over 500: 19.1 and 22.2, over 2000
// (2^29): 45.3 and 32.4; below 64 rows 32 of 8 over 1000: 76.5 and 71.0.
constexpr int k_chunk_rows = 64;                // rows of a sequence on average, at least
constexpr double k_chunk_work = 268435456.0;    // rows x kv heads x cells of the tables x head_dim, at least
// From two tiles of a sequence on the cells are decoded once for all tiles,
// while they fit the workspace.  Measured decoded before and in each workgroup
// (us), 32 heads of 64 and of 128 on 8: 8 sequences of 512 tokens over 2000 cells 214
// and 250, 371 and 430; of 128 tokens (512 rows) 105 and 94, 156 and 149; of 64 tokens
// 69 and 62, 112 and 96; of 32 over 500 32 and 23, 42 and 31.
constexpr int k_decode_rows = 512;
constexpr int64_t k_pre_bytes = (int64_t)1 << 30;   // of the workspace for decoded cells, at most
// Waves of a workgroup.  Up to 64 dims four: two or three workgroups share a CU,
// and uneven sequences leave smaller last tiles (a batch of 9 conversations of
// 5 to 301 tokens 37 us, with eight waves 45, before parts were smaller).  Above, with
// cells decoded before, eight from 2048 rows a sequence on, which copy a cell once for
// 256 rows (one sequence of 4096 tokens behind 4096, 32 heads of 128: 1053 us, with four
// 1104; of 512 rows, 8 of 128 tokens over 2000 cells, 179, with four 157; at the border,
// 4 of 512 tokens, 225 and 200).  Where each workgroup decodes, four, two workgroups
// to a CU, above 128 rows a sequence (8 of 40 tokens over 2000 cells: 77 us, with eight
// 100; of 64: 97 and 122), and eight up to there, of which half decode (32 of 16 over
// 1000: 96 and 76), and for the many rows whose cells the workspace does not hold.
constexpr int k_helped_rows = 128;
constexpr int k_wide_rows = 2048;
// Parts of a row's cells: as many workgroups as a CU runs at a time, a part at
// least so many blocks of 64 cells (single tokens: 64 sequences of up to 8192 cells
// 297 us with 16 a CU, 326 with 4; conversations 33.5 us with parts of 4 blocks, 37.1 with 8
// and 33.1 with 2, of which the join reads more).
constexpr int k_few_wgs = 16, k_few_part = 8, k_many_wgs = 2, k_many_part = 4;
// window: 0, or fewer parts for it (the workspace's size is that without).
static attn_plan plan_attn(const lnship_paged_kv *kv, int64_t rep, int cus, int64_t window) {
    attn_plan p;
    const int64_t rows = kv->ntok * rep, of_seq = kv->n_seq ? rows / kv->n_seq : 0;
    const int64_t n_head = rep * kv->n_head_kv, tile_bytes = kv->n_head_kv * 64 * ((kv->head_dim + 31) & ~(int64_t)31) * 8;
    const int64_t cells = kv->table_ld * kv->page;
    const double work = (double)(rows * kv->n_head_kv) * (double)(cells * kv->head_dim);
    const bool chunks = kv->head_dim <= 128 && of_seq >= k_chunk_rows && work >= k_chunk_work;
    p.pre_tiles = (cells + 63) / 64;
    p.pre = chunks && of_seq >= k_decode_rows && kv->n_seq * p.pre_tiles <= k_pre_bytes / tile_bytes;
    p.pre_bytes = p.pre ? kv->n_seq * p.pre_tiles * tile_bytes : 0;
    p.ok_bytes = p.pre ? (kv->n_seq * p.pre_tiles * 8 + 255) & ~(int64_t)255 : 0;
    p.waves = !chunks ? 0 : kv->head_dim <= 64 || (p.pre ? of_seq < k_wide_rows : of_seq > k_helped_rows && of_seq < k_decode_rows) ? 4 : 8;
    p.tile_rows = p.waves ? p.waves * 32 : 16;
    p.tiles = rows / p.tile_rows + kv->n_seq;
    const int64_t wgs = std::max<int64_t>(1, p.tiles * kv->n_head_kv);
    p.min_per = p.waves ? k_many_part : k_few_part;
    // blocks of 64 cells that a tile sees at most
    const int64_t seen = window > 0 ? std::min(cells, std::min(window, cells) + p.tile_rows / rep + 128) : cells;
    const int64_t most = (seen / 64 + p.min_per - 1) / p.min_per;
    const int64_t want = p.waves ? k_many_wgs : k_few_wgs;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(want * cus + wgs - 1) / wgs, most, 256}));
    p.parts_bytes = p.splits > 1 ? (kv->ntok * n_head * (p.splits * (kv->head_dim + 2) + 1) * 4 + 255) & ~(int64_t)255 : 0;
    return p;
}

// a kernel's LDS limit, set once on a device (done: the devices that know it)
static int allow_lds(const void *kernel, int lds, std::atomic<uint64_t> &done) {
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!(done.load() >> dev & 1)) {
        LNSHIP_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        done.fetch_or((uint64_t)1 << dev);
    }
    return 0;
}

template <int NB, int NW, int C>
static int launch_chunk(const attn_paged_args &m, const dim3 &grid, hipStream_t s, unsigned long long *err) {
    constexpr int lds = 2 * C / 32 * 4 * tile_of<NB>::B * 16;
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_lds(reinterpret_cast<const void *>(k_attn_chunk<NB, NW, C>), lds, done)) return rc;
    hipLaunchKernelGGL((k_attn_chunk<NB, NW, C>), grid, dim3(NW * 64), lds, s, m, err);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

template <int NB>
static int launch_attn(const attn_paged_args &m, const attn_plan &p, int cus, hipStream_t s, unsigned long long *err) {
    if constexpr (NB <= 4) {
        const dim3 chunks((unsigned)(p.tiles * m.kv.n_head_kv), (unsigned)p.splits);
        if (p.pre) {
            // (a grid's y and z are counted in 16 bits)
            const int64_t y = std::min<int64_t>(m.kv.n_seq, 65535 / m.kv.n_head_kv) * m.kv.n_head_kv;
            const int64_t x = std::max<int64_t>(1, std::min<int64_t>(p.pre_tiles, 8 * cus / y));
            hipLaunchKernelGGL(k_attn_decode<NB>, dim3((unsigned)x, (unsigned)y), dim3(256), 0, s, m, err);
            LNSHIP_HIP(hipGetLastError());
            constexpr int most = NB <= 2 ? 4 : 8;
            if (p.waves == 4) hipLaunchKernelGGL((k_attn_tiles<NB, 4>), chunks, dim3(256), 0, s, m, err);
            else hipLaunchKernelGGL((k_attn_tiles<NB, most>), chunks, dim3(most * 64), 0, s, m, err);
            LNSHIP_HIP(hipGetLastError());
            return 0;
        }
        if (p.waves == 4) return launch_chunk<NB, 4, NB <= 2 ? 64 : 32>(m, chunks, s, err);
        if constexpr (NB > 2)
            if (p.waves == 8) return launch_chunk<NB, 8, 64>(m, chunks, s, err);
    }
    const dim3 grid((unsigned)p.tiles, (unsigned)m.kv.n_head_kv, (unsigned)p.splits);
    // A CU for each workgroup: eight waves, which go over their cells in half the steps
    // (448 cells of 9 heads of 64 on 3 11.0 us, with four 12.1; 32 heads of 128 on 8 17.4
    // and 18.9; 64 sequences of 2000 cells of those 167 with eight, 129 with four).
    if constexpr (NB <= 4)
        if (p.tiles * m.kv.n_head_kv * p.splits <= cus) {
            if (m.kv.head_dim == NB * 32) hipLaunchKernelGGL((k_attn_paged<NB, true, 8>), grid, dim3(512), 0, s, m, err);
            else hipLaunchKernelGGL((k_attn_paged<NB, false, 8>), grid, dim3(512), 0, s, m, err);
            LNSHIP_HIP(hipGetLastError());
            return 0;
        }
    if (m.kv.head_dim == NB * 32) hipLaunchKernelGGL((k_attn_paged<NB, true, 4>), grid, dim3(256), 0, s, m, err);
    else hipLaunchKernelGGL((k_attn_paged<NB, false, 4>), grid, dim3(256), 0, s, m, err);
    LNSHIP_HIP(hipGetLastError());
    return 0;
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
    if (!a->k || !a->v || (a->n_head && (!a->q || !a->q_dst)) || (a->rope_n_dims && a->n_pos && !a->cos_sin))
        return fail(LNSHIP_EINVAL, "rope_store_kv_paged: null pointer%s");
    if (a->n_head && !same_or_apart(a->q, a->q_ld, a->q_dst, s.a.q_dst_ld, nq, kv->ntok))
        return fail(LNSHIP_EINVAL, "rope_store_kv_paged: q_dst overlaps q%s");
    device_state *st = state();
    if (!st) return LNSHIP_ENOINIT;
    // 16-byte loads and stores, and eight dims a thread
    const bool vec = a->rope_n_dims > 0 && a->rope_n_dims % 8 == 0 &&
                     (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->cos_sin | (uintptr_t)a->q_dst) & 15) == 0 &&
                     ((a->q_ld | a->k_ld | s.a.q_dst_ld) & 3) == 0;
    // (its tables take 4 us to lay out: 64 rows of 32 heads of 128 on 8 6.3 us without,
    // 8.5 so, 128 rows 8.5 and 8.9, 256 13.8 and 10.2; 128 of 9 heads of 64 on 3 4.9 and 8.4)
    if (vec && nq <= 1 << 26 && kv->ntok * (nq + 2 * nk) >= 1 << 19) {
        // Eight rows of a prompt together, as their cells share cache lines (8 prompts
        // of 1400 tokens, 32 heads of 64 on 8: 68 us, by single rows 80); single
        // tokens' rows, and few, by themselves (4096 sequences' tokens, heads of 128: 75,
        // by eight 83).  Workgroups: 16 a CU, if there is an item for each thread (256
        // tokens 10.2 us, a workgroup a row 13.2).
        const int sh = kv->ntok >= 1024 && kv->ntok >= 8 * kv->n_seq ? 3 : 0;
        const int64_t x = (((kv->ntok + (1 << sh) - 1) >> sh) + 7) / 8 * 8;   // (all of every XCD's share)
        const int64_t items = (nq / 8 + nk / 8 + nk / 4) << sh;
        const int64_t y = std::max<int64_t>(1, std::min(16 * st->cus / x, items / k_block));
        const dim3 grid((unsigned)x, (unsigned)y);
        if (a->neox) hipLaunchKernelGGL(k_store_paged_rows<true>, grid, dim3(k_block), 0, (hipStream_t)stream, s, sh, st->T, st->index_err);
        else hipLaunchKernelGGL(k_store_paged_rows<false>, grid, dim3(k_block), 0, (hipStream_t)stream, s, sh, st->T, st->index_err);
        LNSHIP_HIP(hipGetLastError());
        return 0;
    }
    const int64_t items = (a->n_head + kv->n_head_kv) * (kv->head_dim - a->rope_n_dims / 2) + nk;
    const int64_t y = std::min<int64_t>((items + k_block - 1) / k_block, 65535);
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
    const attn_plan p = plan_attn(kv, n_head / kv->n_head_kv, st->cus, 0);
    return p.parts_bytes + p.pre_bytes + p.ok_bytes;
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
    if (!same_or_apart(a->q, q_ld, a->dst, dst_ld, nq, kv->ntok))
        return fail(LNSHIP_EINVAL, "attn_paged: dst overlaps q%s");
    device_state *st = state();
    if (!st) return LNSHIP_ENOINIT;
    const int64_t rep = a->n_head / kv->n_head_kv;
    const attn_plan p = plan_attn(kv, rep, st->cus, a->window);
    const int64_t need = p.parts_bytes + p.pre_bytes + p.ok_bytes;
    if (need && (!a->work || a->work_bytes < (size_t)need || ((uintptr_t)a->work & 15)))
        return fail(LNSHIP_EINVAL, "attn_paged: work smaller than lnship16_attn_paged_work or not aligned%s");
    // (a grid's threads along x are counted in 32 bits)
    if (kv->ntok * rep > 0xfffffff || p.tiles * kv->n_head_kv > 0x7fffff || kv->ntok * a->n_head > 0xffffff)
        return fail(LNSHIP_ERANGE, "attn_paged: grid too large%s");
    attn_paged_args m{*kv, a->q, a->dst, q_ld, dst_ld, a->scale * 1.44269504088896341f,
                      a->window > 0x3fffffff ? 0 : (int)a->window, (int)a->n_head, (int)rep, log2_of(kv->page), p.splits,
                      p.tile_rows, p.min_per, q_ld % 4 == 0 && ((uintptr_t)a->q & 15) == 0};
    const int64_t all = kv->ntok * a->n_head;
    char *work = (char *)a->work;
    if (p.splits > 1) {
        m.sums = (float *)work;
        m.stats = (float2 *)(m.sums + p.splits * all * kv->head_dim);
        m.used = (int *)(m.stats + p.splits * all);
    }
    if (p.pre) {
        m.pre = (uint4 *)(work + p.parts_bytes);
        m.pre_ok = (uint8_t *)(work + p.parts_bytes + p.pre_bytes);
        m.pre_tiles = (int)p.pre_tiles;
    }
    if (kv->n_pages == 0) m.kv.table_ld = 0;   // no page to read: no cells
    hipStream_t s = (hipStream_t)stream;
    int rc;
    switch ((kv->head_dim + 31) / 32) {
        case 1: rc = launch_attn<1>(m, p, st->cus, s, st->index_err); break;
        case 2: rc = launch_attn<2>(m, p, st->cus, s, st->index_err); break;
        case 3: rc = launch_attn<3>(m, p, st->cus, s, st->index_err); break;
        case 4: rc = launch_attn<4>(m, p, st->cus, s, st->index_err); break;
        case 5: rc = launch_attn<5>(m, p, st->cus, s, st->index_err); break;
        case 6: rc = launch_attn<6>(m, p, st->cus, s, st->index_err); break;
        case 7: rc = launch_attn<7>(m, p, st->cus, s, st->index_err); break;
        default: rc = launch_attn<8>(m, p, st->cus, s, st->index_err);
    }
    if (rc || p.splits == 1) return rc;
    if (p.splits > 8) hipLaunchKernelGGL(k_attn_paged_join<4>, dim3((unsigned)all), dim3(256), 0, s, m);
    else hipLaunchKernelGGL(k_attn_paged_join<1>, dim3((unsigned)((all + 3) / 4)), dim3(256), 0, s, m);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
