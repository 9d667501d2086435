// Drawing tokens from rows of logits: temperature, top-k, top-p, min-p and a
// given uniform random number (include/lnship.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lnship.h"
#include "lnship_device.h"
#include "lnship_host.h"

namespace lnship {

#ifndef LNSHIP_RES
#define LNSHIP_RES 3
#endif
constexpr int k_draw_block = 1024;
constexpr int k_draw_waves = k_draw_block / 64;
constexpr int k_w_sh = 40;              // weights are integers in units of 2^-40
constexpr int k_seg = 1024;             // logits of a segment, which a wave goes through at a time
constexpr int k_seg_max = 512;
constexpr int64_t k_draw_vocab = (int64_t)k_seg * k_seg_max;
constexpr int k_bins = 4096, k_bins_binade = 64;   // of the distance from the largest logit, 64 a binade of weight
constexpr int k_list = 2048;            // tokens that are put in order at once
constexpr int k_small_k = 1024;         // a top_k whose tokens are

// a key that orders floats: NaN lowest, then -inf up; -0 equal to 0
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = f32_bits(x + 0.0f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t k_key_ninf = 0x007fffffu;   // order_key(-inf)

// The weight e^((x - x_max) / T) in units of 2^-40, rounded.  The exponent is
// formed in 64 bits (32 would lose what tells two sums apart), its fraction's
// power in 32: 24 bits of every weight.  Integers come out of the low bits of
// a sum with a power of two, which costs less than a conversion: 17 issue slots
// a weight, four of them the power.
struct weigher {
    double xmax, f;   // f = log2 e / T
    __device__ __forceinline__ uint64_t operator()(float x) const {
        constexpr double whole = 6755399441055744.0;   // 1.5 2^52: a sum's low word is the integer
        constexpr double unit = 4096.0;                // a sum's last place is 2^-40
        const double y = fmax(((double)x - xmax) * f, -63.0);   // (-inf times an f of 0: -63)
        const double t = y + whole;
        // 2^r in [2^-1/2, 2^1/2]
        const float p = __builtin_amdgcn_exp2f((float)(y - (t - whole)));
        const double w = ldexp((double)p, (int)(uint32_t)__double_as_longlong(t));
        return (uint64_t)__double_as_longlong(w + unit) - (uint64_t)__double_as_longlong(unit);
    }
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

struct draw_args {
    const float *logits;
    int64_t ld;
    int n;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int32_t *tokens;
    float *probs;
};

struct draw_row {   // what a row asks for
    float xmax;
    weigher W;
    int top_k;      // 0: no limit
    float top_p;
    double wmin;    // least weight that min_p keeps, in units
};

// the unit of the total that u names
__device__ __forceinline__ uint64_t draw_target(float u, uint64_t total) {
    const double at = u > 0.0f ? (double)u * (double)total : 0.0;
    return at >= (double)total ? total - 1 : min((uint64_t)at, total - 1);
}

// inclusive sums over the workgroup's threads; the same memory may be used
// again after the next barrier
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *s, uint64_t &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    if (lane == 63) s[wave] = v;
    __syncthreads();
    uint64_t t = lane < k_draw_waves ? s[lane] : 0;
    for (int d = 1; d < k_draw_waves; d <<= 1) {
        const uint64_t o = __shfl_up(t, d);
        if (lane >= d) t += o;
    }
    all = __shfl(t, k_draw_waves - 1);
    const uint64_t before = __shfl(t, max(wave - 1, 0));
    return wave ? v + before : v;
}

// The items of list (all different) put in descending order: each item's place
// is the number of larger ones, counted by as many threads as there are for
// an item.  m <= k_list; list and out apart; ends with a barrier.  A thread
// reads the items that lie `of` apart, so that a wave's reads are one address.
__device__ __forceinline__ void order_items(const uint64_t *list, uint64_t *out, uint32_t *place, int m) {
    for (int i = threadIdx.x; i < m; i += k_draw_block) place[i] = 0;
    __syncthreads();
    int sh = 0;   // 2^sh items a turn, the block's other threads beside them
    while ((64 << sh) < m && (64 << sh) < k_draw_block) sh++;
    const int width = 64 << sh, of = k_draw_block / width, part = threadIdx.x / width;
    for (int i = threadIdx.x & (width - 1); i < m; i += width) {
        const uint64_t own = list[i];
        uint32_t c = 0;
#pragma unroll 4
        for (int j = part; j < m; j += of) c += list[j] > own;
        if (of == 1) place[i] = c;
        else atomicAdd(&place[i], c);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += k_draw_block) out[place[i]] = list[i];
    __syncthreads();
}

// Any row, in passes over the memory: the border of the top_k first, then that
// of top_p, digit by digit of the ordered keys, over a histogram of counts or
// weights of the keys that have the digits so far; ties at a border are kept
// from the lowest index on.  For rows that k_draw's one histogram does not
// resolve: thousands of equal logits at a border, a large top_k, infinities.
__device__ __forceinline__ void draw_by_digits(const draw_args &a, const draw_row &d0, int64_t r, uint64_t *s_w,
                                                         uint64_t *s_u64) {
    __shared__ uint32_t s_c[256], s_u32[k_draw_waves], s_digit;
    __shared__ uint64_t s_above_w;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
    const float *x = a.logits + r * a.ld;
    // (an infinite largest logit, or 1 / T: only its equals weigh anything)
    const bool sharp = !(fabsf(d0.xmax) < INFINITY) || !(d0.W.f < 1e300);
    auto W = [&](float v) { return sharp ? (uint64_t)(v == d0.xmax) << k_w_sh : d0.W(v); };
    const int top_k = d0.top_k;
    const float top_p = d0.top_p;
    const double wmin = d0.wmin;
    __syncthreads();   // (what lay in s_w and s_u64 is read)
    // the border key and how many of its ties are kept
    uint32_t bkey = k_key_ninf + 1, bties = 0xffffffffu;
    // by_count: the key of rank want (from 1), else the key where the weights'
    // sum reaches want; over keys above `bkey` and its first bties
    auto select = [&](bool by_count, uint64_t want) {
        uint32_t key = 0;
        uint64_t above = 0;
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int i = tid; i < 256; i += k_draw_block) {
                s_w[i] = 0;
                s_c[i] = 0;
            }
            __syncthreads();
            for (int i = tid; i < n; i += k_draw_block) {
                const float v = x[i];
                const uint32_t k = order_key(v);
                if (k < bkey || (sh < 24 && (k >> (sh + 8)) != (key >> (sh + 8)))) continue;
                const uint32_t d = (k >> sh) & 255u;
                if (by_count) {
                    atomicAdd(&s_c[d], 1u);
                } else if (k != bkey || bties == 0xffffffffu) {
                    atomicAdd((unsigned long long *)&s_w[d], (unsigned long long)W(v));
                }
            }
            if (!by_count && bties != 0xffffffffu && tid == 0 && (sh == 24 || (bkey >> (sh + 8)) == (key >> (sh + 8))))
                atomicAdd((unsigned long long *)&s_w[(bkey >> sh) & 255u],
                          (unsigned long long)(W(key_value(bkey)) * bties));
            __syncthreads();
            if (tid == 0) {
                uint64_t sum = above;
                int d = 255;
                for (; d > 0; d--) {
                    const uint64_t v = by_count ? (uint64_t)s_c[d] : s_w[d];
                    if (sum + v >= want) break;
                    sum += v;
                }
                s_digit = (uint32_t)d;
                s_above_w = sum;
            }
            __syncthreads();
            key |= s_digit << sh;
            above = s_above_w;
            __syncthreads();
        }
        const uint64_t rest = want - above;   // of the border key
        if (by_count) {
            bkey = key;
            bties = (uint32_t)rest;
        } else {
            const uint64_t w = max(W(key_value(key)), (uint64_t)1);
            const uint64_t need = (rest + w - 1) / w;
            if (key != bkey) bties = 0xffffffffu;
            bkey = key;
            bties = (uint32_t)min((uint64_t)bties, need);
        }
    };
    auto block_sum = [&](uint64_t v) {
        v = wave_sum(v);
        if (lane == 0) s_u64[wave] = v;
        __syncthreads();
        uint64_t t = 0;
        for (int w = 0; w < k_draw_waves; w++) t += s_u64[w];
        __syncthreads();
        return t;
    };

    if (top_k > 0 && top_k < n) {
        // (fewer logits above -inf than top_k: no border)
        uint64_t c = 0;
        for (int i = tid; i < n; i += k_draw_block) c += order_key(x[i]) > k_key_ninf;
        if (block_sum(c) > (uint64_t)top_k) select(true, (uint64_t)top_k);
    }
    if (top_p < 1.0f) {
        uint64_t w = 0;
        for (int i = tid; i < n; i += k_draw_block) {
            const float v = x[i];
            const uint32_t k = order_key(v);
            if (k > bkey || (k == bkey && bties == 0xffffffffu)) w += W(v);
        }
        w = block_sum(w);
        if (bties != 0xffffffffu) w += W(key_value(bkey)) * bties;
        const double want = ceil((double)top_p * (double)w);
        select(false, want >= 1.0 ? min((uint64_t)want, w) : (uint64_t)1);
    }

    // the kept weights' sum, then the token: blocks of the row in order, each
    // thread one token; equal keys at the border counted in order
    auto pass = [&](uint64_t target, bool draw, uint64_t &total) {
        uint64_t run = 0;
        uint32_t ties = 0;
        for (int i0 = 0; i0 < n; i0 += k_draw_block) {
            const int i = i0 + tid;
            const float v = i < n ? x[i] : -INFINITY;
            const uint32_t k = order_key(v);
            uint64_t w = 0;
            bool keep = k > bkey;
            if (bties != 0xffffffffu) {
                const uint64_t eq = __ballot(k == bkey);
                if (lane == 0) s_u32[wave] = (uint32_t)__popcll(eq);
                __syncthreads();
                uint32_t before = ties, all = ties;
                for (int q = 0; q < k_draw_waves; q++) {
                    if (q < wave) before += s_u32[q];
                    all += s_u32[q];
                }
                before += (uint32_t)__popcll(eq & (((uint64_t)1 << lane) - 1));
                ties = all;
                keep |= k == bkey && before < bties;
                __syncthreads();
            } else {
                keep |= k == bkey;
            }
            if (keep) {
                w = W(v);
                if ((double)w < wmin) w = 0;
            }
            if (!draw) {
                run += w;
                continue;
            }
            uint64_t inc = w;
            for (int d = 1; d < 64; d <<= 1) {
                const uint64_t o = __shfl_up(inc, d);
                if (lane >= d) inc += o;
            }
            if (lane == 63) s_u64[wave] = inc;
            __syncthreads();
            uint64_t all = 0, before = run;
            for (int q = 0; q < k_draw_waves; q++) {
                if (q < wave) before += s_u64[q];
                all += s_u64[q];
            }
            if (before + inc > target && before + inc - w <= target) {
                a.tokens[r] = i;
                if (a.probs) a.probs[r] = (float)((double)w / (double)total);
            }
            run += all;
            __syncthreads();
            if (run > target) return;
        }
        if (!draw) total = block_sum(run);
    };
    uint64_t total = 0;
    pass(0, false, total);
    pass(draw_target(a.u[r], total), true, total);
}

// One workgroup a row; a wave goes through segments of 1024 logits.  R segments
// a wave are held in registers; the rest of a longer row (MORE) is read again
// for every pass.
// After its largest logit is known:
// - without top_k and top_p the weights are summed by segment, the segment that
//   holds u's share found, and that segment gone through again;
// - with them one histogram over the distance from the largest logit (of counts
//   for top_k, of weights for top_p) names the bin of the border; with a top_k
//   the tokens down to that bin, with top_p alone those of that bin, are
//   put in order, and the border is exact.
template <int R, bool MORE>
__global__ __launch_bounds__(k_draw_block) void k_draw(draw_args a) {
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // rows need no alignment
    __shared__ uint64_t s_hist[k_bins];   // later the lists
    __shared__ uint64_t s_seg[k_list / 2];   // segments' sums; before, the places of order_items
    static_assert(k_seg_max <= k_list / 2, "");
    __shared__ uint64_t s_scan[2][k_draw_waves];
    __shared__ uint64_t s_x[2];
    __shared__ int s_n;
    uint64_t *const s_list = s_hist, *const s_sorted = s_hist + k_list;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n, segs = (n + k_seg - 1) / k_seg;
    const int64_t r = blockIdx.x;
    const float *x = a.logits + r * a.ld;
    static_assert(2 * k_list <= k_bins, "both lists lie in the histogram's place");

    // a segment's sixteen logits of a lane, v[4 q + j] number 256 q + 4 lane + j;
    // NaN, and what lies past the row, as -inf
    auto load = [&](int seg, float (&v)[16]) {
        const int i0 = seg * k_seg + lane * 4;
        if ((seg + 1) * k_seg <= n) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float4u t = *reinterpret_cast<const float4u *>(x + i0 + 256 * q);
                v[4 * q] = t[0], v[4 * q + 1] = t[1], v[4 * q + 2] = t[2], v[4 * q + 3] = t[3];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int i = i0 + (e >> 2) * 256 + (e & 3);
                const float t = x[min(i, n - 1)];
                v[e] = i < n ? t : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = fmaxf(v[e], -INFINITY);
    };
    auto index = [&](int seg, int e) { return seg * k_seg + (e >> 2) * 256 + lane * 4 + (e & 3); };
    // f(segment, its logits) for every segment of the wave: the first R are kept
    // in registers, the others loaded for every pass, one ahead
    float keep[R][16];
#pragma unroll
    for (int i = 0; i < R; i++)
        if (i * k_draw_waves + wave < segs) load(i * k_draw_waves + wave, keep[i]);
    auto each = [&](auto f) {
        float next[16];
        int seg = R * k_draw_waves + wave;
        if (MORE && seg < segs) load(seg, next);
#pragma unroll
        for (int i = 0; i < R; i++)
            if (i * k_draw_waves + wave < segs) f(i * k_draw_waves + wave, keep[i]);
        if constexpr (MORE)
            for (; seg < segs; seg += k_draw_waves) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = next[e];
                if (seg + k_draw_waves < segs) load(seg + k_draw_waves, next);
                f(seg, v);
            }
    };

    draw_row D;
    auto easy = [&]() -> bool {
        // the largest logit, and the first index that has it
        const float T = a.temperature ? a.temperature[r] : 1.0f;
        const bool greedy = !(T > 0.0f);
        float mx = -INFINITY;
        int at = 0x7fffffff;
        if (!greedy) {
            each([&](int, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, v[e]);
            });
        } else {
            each([&](int seg, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                        if (v[e] > mx) {
                            mx = v[e];
                            at = index(seg, e);
                        }
            });
        }
        uint64_t best = (uint64_t)order_key(mx) << 32 | (uint32_t)(0x7fffffff - at);
        for (int d = 32; d; d >>= 1) best = max(best, (uint64_t)__shfl_xor(best, d));
        if (lane == 0) s_scan[0][wave] = best;
        __syncthreads();
        best = s_scan[0][lane & (k_draw_waves - 1)];
        for (int d = k_draw_waves / 2; d; d >>= 1) best = max(best, (uint64_t)__shfl_xor(best, d));
        const uint32_t kmax = (uint32_t)(best >> 32);
        if (kmax <= k_key_ninf || greedy) {
            if (tid == 0) {
                a.tokens[r] = kmax <= k_key_ninf ? -1 : 0x7fffffff - (int32_t)(uint32_t)best;
                if (a.probs) a.probs[r] = kmax <= k_key_ninf ? 0.0f : 1.0f;
            }
            return true;
        }
        D.xmax = key_value(kmax);
        D.W = {(double)D.xmax, 1.4426950408889634 / (double)T};
        D.top_k = a.top_k ? a.top_k[r] : 0;
        if (D.top_k < 0 || D.top_k >= n) D.top_k = 0;
        D.top_p = a.top_p ? a.top_p[r] : 1.0f;
        if (!(D.top_p < 1.0f)) D.top_p = 1.0f;
        // (the largest logit weighs 2^40 units)
        const float min_p = a.min_p ? a.min_p[r] : 0.0f;
        D.wmin = min_p > 0.0f ? fmin((double)min_p, 1.0) * (double)((uint64_t)1 << k_w_sh) : 0.0;
        const weigher &W = D.W;
        const bool by_count = D.top_k > 0;
        const float scale = (float)(k_bins_binade * D.W.f);
        if (D.top_k > k_small_k || !(fabsf(D.xmax) < INFINITY) || !(scale < INFINITY)) {
            return false;
        }

        // a token is kept if (key, index) does not come behind (bkey, bidx)
        uint32_t bkey = 0;
        int bidx = 0x7fffffff, above_bin = k_bins;
        if (by_count || D.top_p < 1.0f) {
            // bin of a logit: it never rises with the logit; the last holds all
            // whose weight rounds to 0
            auto bin_of = [&](float v) { return (int)fminf((D.xmax - v) * scale, (float)(k_bins - 1)); };
            for (int i = tid; i < k_bins; i += k_draw_block) s_hist[i] = 0;
            if (tid == 0) s_n = 0;
            __syncthreads();
            if (by_count) {
                each([&](int, const float *v) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                            const int b = bin_of(v[e]);
                            if (b < k_bins - 1) atomicAdd((unsigned int *)&s_hist[b], 1u);
                        }
                });
            } else {
                each([&](int, const float *v) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                            const int b = bin_of(v[e]);
                            if (b < k_bins - 1) atomicAdd((unsigned long long *)&s_hist[b], (unsigned long long)W(v[e]));
                        }
                });
            }
            __syncthreads();
            // the first bin up to which the counts (the weights) reach what is kept
            uint64_t h[4], sum = 0, all;
#pragma unroll
            for (int i = 0; i < 4; i++) sum += h[i] = s_hist[tid * 4 + i];
            uint64_t run = block_scan(sum, s_scan[1], all) - sum;
            uint64_t want = (uint64_t)D.top_k;
            if (!by_count) {
                const double p = ceil((double)D.top_p * (double)all);
                want = p >= 1.0 ? min((uint64_t)p, all) : 1;
            }
            if (tid == 0) s_x[0] = k_bins - 1;   // (top_k: fewer weigh anything)
            __syncthreads();
            if (run < want && run + sum >= want) {
                int b = tid * 4;
#pragma unroll
                for (int i = 0; i < 3; i++)
                    if (run + h[i] < want) run += h[i], b++;
                    else break;
                s_x[0] = (uint64_t)b;
                s_x[1] = run;
            }
            __syncthreads();   // (the histogram is read; its place is the lists')
            const int border = (int)s_x[0];
            if (border < k_bins - 1) {
                const uint64_t above = s_x[1];
                const int from = by_count ? 0 : border;   // the bins of the list
                each([&](int seg, const float *v) {
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                            const int b = bin_of(v[e]);
                            if (b <= border && b >= from) {
                                const int i = atomicAdd(&s_n, 1);
                                if (i < k_list)
                                    s_list[i] = (uint64_t)order_key(v[e]) << 32 |
                                                (uint32_t)(0x7fffffff - index(seg, e));
                            }
                        }
                });
                __syncthreads();
                const int m = s_n;
                if (m > k_list) {
                    return false;
                }
                uint32_t *const place = (uint32_t *)s_seg;
                order_items(s_list, s_sorted, place, m);
                if (by_count) {
                    // the first top_k, of those top_p's, of those min_p's; then by index
                    const int k = min(D.top_k, m);
                    uint64_t w = tid < k ? W(key_value((uint32_t)(s_sorted[tid] >> 32))) : 0, total;
                    uint64_t c = block_scan(w, s_scan[0], total);
                    int kept = k;
                    if (D.top_p < 1.0f) {
                        const double p = ceil((double)D.top_p * (double)total);
                        const uint64_t need = p >= 1.0 ? min((uint64_t)p, total) : 1;
                        if (tid == 0) s_n = 1;
                        __syncthreads();
                        if (tid < k && c - w < need && c >= need) s_n = tid + 1;
                        __syncthreads();
                        kept = s_n;
                    }
                    const bool in = tid < kept && w > 0 && (double)w >= D.wmin;
                    if (tid < k_list / 2) s_list[tid] = 0;   // (what is not kept comes last)
                    __syncthreads();
                    // order by index: its complement above, its place in the ranking below
                    if (tid < kept) s_list[tid] = (uint64_t)(uint32_t)s_sorted[tid] << 32 | (in ? (uint32_t)tid + 1u : 0u);
                    __syncthreads();
                    uint64_t *const by_index = s_sorted + k_list / 2;   // (top_k <= k_list / 2)
                    order_items(s_list, by_index, place, kept);
                    const uint32_t rank = tid < kept ? (uint32_t)by_index[tid] : 0u;
                    const uint64_t item = rank ? s_sorted[rank - 1] : 0;
                    w = rank ? W(key_value((uint32_t)(item >> 32))) : 0;
                    c = block_scan(w, s_scan[1], total);
                    const uint64_t target = draw_target(a.u[r], total);
                    if (w && c > target && c - w <= target) {
                        a.tokens[r] = 0x7fffffff - (int32_t)(uint32_t)item;
                        if (a.probs) a.probs[r] = (float)((double)w / (double)total);
                    }
                    return true;
                }
                // top_p: the border bin's first, as many as the weight still needs
                if (tid == 0) s_n = m;
                __syncthreads();
                uint64_t before = above;
                for (int i0 = 0; i0 < m; i0 += k_draw_block) {
                    uint64_t part;
                    const uint64_t w = i0 + tid < m ? W(key_value((uint32_t)(s_sorted[i0 + tid] >> 32))) : 0;
                    const uint64_t c = before + block_scan(w, s_scan[(i0 / k_draw_block) & 1], part);
                    if (c - w < want && c >= want) s_n = i0 + tid + 1;
                    before += part;
                }
                __syncthreads();
                const uint64_t item = s_sorted[s_n - 1];
                bkey = (uint32_t)(item >> 32);
                bidx = 0x7fffffff - (int)(uint32_t)item;
                above_bin = border;
                __syncthreads();
            }
        }
        auto weigh = [&](float v, int i) {
            uint64_t w = W(v);
            if ((double)w < D.wmin) w = 0;
            if (above_bin < k_bins) {
                const uint32_t k = order_key(v);
                if (k < bkey || (k == bkey && i > bidx)) w = 0;
            }
            return w;
        };
        each([&](int seg, const float *v) {
            uint64_t w = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) w += weigh(v[e], index(seg, e));
            w = wave_sum(w);
            if (lane == 0) s_seg[seg] = w;
        });
        __syncthreads();
        uint64_t total;
        const uint64_t w = tid < segs ? s_seg[tid] : 0, c = block_scan(w, s_scan[0], total);
        const uint64_t target = draw_target(a.u[r], total);
        if (c > target && c - w <= target) {
            s_n = tid;
            s_x[0] = target - (c - w);
        }
        __syncthreads();
        // the segment's tokens, one a thread
        const int i = s_n * k_seg + tid;
        const uint64_t left = s_x[0];
        const float v = i < n ? x[i] : -INFINITY;
        const uint64_t wi = i < n && v == v ? weigh(v, i) : 0;
        uint64_t of_seg;
        const uint64_t ci = block_scan(wi, s_scan[1], of_seg);
        if (ci > left && ci - wi <= left) {
            a.tokens[r] = i;
            if (a.probs) a.probs[r] = (float)((double)wi / (double)total);
        }
        return true;
    };
    if (!easy()) draw_by_digits(a, D, r, s_hist, s_scan[0]);
}

}  // namespace lnship

using namespace lnship;

extern "C" {

int64_t lnship_sample_work(int64_t n_rows, int64_t n_vocab) {
    if (n_rows < 0 || n_vocab < 0) return fail(LNSHIP_EINVAL, "sample: bad shape%s");
    if (n_rows > 0x3fffff || n_vocab > k_draw_vocab) return fail(LNSHIP_ERANGE, "sample: too large%s");
    return 0;
}

int lnship_sample(const lnship_sample_args *a, void *stream) {
    if (!a) return fail(LNSHIP_EINVAL, "sample: null arguments%s");
    const int64_t need = lnship_sample_work(a->n_rows, a->n_vocab);
    if (need < 0) return (int)need;
    const int64_t ld = a->ld ? a->ld : a->n_vocab;
    if (a->n_vocab < 1 || ld < a->n_vocab) return fail(LNSHIP_EINVAL, "sample: bad shape%s");
    if (a->n_rows == 0) return 0;
    if (!a->logits || !a->u || !a->tokens) return fail(LNSHIP_EINVAL, "sample: null pointer%s");
    if (need && (!a->work || a->work_bytes < (size_t)need || ((uintptr_t)a->work & 15)))
        return fail(LNSHIP_EINVAL, "sample: work smaller than lnship_sample_work or not aligned%s");
    device_state *s = state();
    if (!s) return LNSHIP_ENOINIT;
    draw_args d{a->logits, ld, (int)a->n_vocab, a->temperature, a->top_k, a->top_p, a->min_p, a->u, a->tokens, a->probs};
    const dim3 grid((unsigned)a->n_rows), block(k_draw_block);
    hipStream_t st = (hipStream_t)stream;
    const int rounds = (int)((a->n_vocab + k_seg * k_draw_waves - 1) / (k_seg * k_draw_waves));
    if (rounds == 1) hipLaunchKernelGGL((k_draw<1, false>), grid, block, 0, st, d);
    else if (rounds == 2) hipLaunchKernelGGL((k_draw<2, false>), grid, block, 0, st, d);
    else if (rounds == 3) hipLaunchKernelGGL((k_draw<3, false>), grid, block, 0, st, d);
    else hipLaunchKernelGGL((k_draw<LNSHIP_RES, true>), grid, block, 0, st, d);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
