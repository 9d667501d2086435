// Drawing tokens from rows of logits: temperature, top-k, top-p, min-p and a
// given uniform random number (include/lnship.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lnship.h"
#include "lnship_device.h"
#include "lnship_host.h"

namespace lnship {

constexpr int k_draw_block = 1024;
constexpr int k_draw_waves = k_draw_block / 64;
constexpr int k_w_sh = 40;              // weights are integers in units of 2^-40
constexpr int k_seg = 1024;             // logits of a segment, which a wave goes through at a time
constexpr int k_seg_max = 512;
constexpr int64_t k_draw_vocab = (int64_t)k_seg * k_seg_max;
constexpr int k_bins = 4096, k_bins_binade = 64;   // of the distance from the largest logit, 64 a binade of weight
constexpr int k_head = 22 * k_bins_binade;   // bins above those of 42 binades, for logits above the first ones
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

// a value that is the same in all lanes, in scalar registers
template <class V>
__device__ __forceinline__ V uniform(V v) {
    union {
        V v;
        int w[sizeof(V) / 4];
    } u;
    u.v = v;
    for (size_t i = 0; i < sizeof(V) / 4; i++) u.w[i] = __builtin_amdgcn_readfirstlane(u.w[i]);
    return u.v;
}

// 2^r for r in [-1/2, 1/2], to 2^-34: the polynomial of degree 7 through it at the
// Chebyshev nodes of that range.
__device__ __forceinline__ double power(double r) {
    double p = 1.5303700711425663e-05;
    p = fma(p, r, 0.00015469729214122798);
    p = fma(p, r, 0.0013333478473685175);
    p = fma(p, r, 0.009618025613318018);
    p = fma(p, r, 0.055504109063258665);
    p = fma(p, r, 0.24022651213498092);
    p = fma(p, r, 0.6931471805568324);
    return fma(p, r, 0.9999999999595618);
}

// 2^y, y in [-64, 0], in units of 2^-40, rounded.  A sum with a power of two
// splits y and makes the result an integer, which costs less than conversions;
// the whole part goes into the power's exponent.  All in 64 bits: in 32 the
// weights of a few likely tokens are off by more than the share of a token of a
// large vocabulary's tail, and another than it would be drawn now and then.
__device__ __forceinline__ uint64_t in_units(double y) {
    constexpr double whole = 6755399441055744.0;   // 1.5 2^52: a sum's low word is the integer
    constexpr double unit = 4096.0;                // a sum's last place is 2^-40
    const double t = y + whole;
    const uint64_t p = (uint64_t)__double_as_longlong(power(y - (t - whole)));
    const uint32_t hi = (uint32_t)(p >> 32) + ((uint32_t)(uint64_t)__double_as_longlong(t) << 20);
    const double w = __longlong_as_double((int64_t)((uint64_t)hi << 32 | (uint32_t)p));
    return (uint64_t)__double_as_longlong(w + unit) - (uint64_t)__double_as_longlong(unit);
}

// The weight e^((x - x_max) / T) in units of 2^-40, of any x_max and T.
struct any_weigher {
    double xmax, f;   // f = log2 e / T
    __device__ __forceinline__ uint64_t operator()(float x) const {
        return in_units(fmax(((double)x - xmax) * f, -63.0));   // (-inf times an f of 0: -63)
    }
};

// The same where |x_max f| <= 2^20: the exponent in one product, to 2^-33.  Some 105
// cycles of a wave, most of them the 13 operations of 64 bits.
struct weigher {
    double f, c;
    float lo;   // x where the weight is 2^-63: what lies below weighs nothing either
    static __device__ __forceinline__ bool fits(float xmax, double f) {
        return fabs((double)xmax * f) <= 1048576.0 && f >= 1e-30;
    }
    __device__ __forceinline__ weigher(float xmax, double f_)
        : f(f_), c(uniform(-(double)xmax * f_)), lo(uniform((float)fmax((double)xmax - 63.0 / f_, -3.4028234e38))) {}
    __device__ __forceinline__ uint64_t operator()(float x) const { return in_units(fma((double)fmaxf(x, lo), f, c)); }
};

// v of the lane that DPP control C names, in the rows of M; zero where there is none
template <int C, int M = 0xf>
__device__ __forceinline__ uint64_t lane_of(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, C, M, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), C, M, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// Inclusive scans over a row's 16 lanes, and the wave's 64: shifts by 1, 2, 4, 8
// within rows, then the last lanes of rows 0 and 2, then of the lower half, added
// to what lies behind.  From register to register: through LDS's permutation a
// step takes as long as five of these.
template <class F>
__device__ __forceinline__ uint64_t row_scan(uint64_t v, F f) {
    v = f(v, lane_of<0x111>(v));
    v = f(v, lane_of<0x112>(v));
    v = f(v, lane_of<0x114>(v));
    return f(v, lane_of<0x118>(v));
}
template <class F>
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, F f) {
    v = row_scan(v, f);
    v = f(v, lane_of<0x142, 0xa>(v));
    return f(v, lane_of<0x143, 0xc>(v));
}
struct add_u64 {
    __device__ __forceinline__ uint64_t operator()(uint64_t x, uint64_t y) const { return x + y; }
};
struct max_u64 {
    __device__ __forceinline__ uint64_t operator()(uint64_t x, uint64_t y) const { return max(x, y); }
};
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return read_lane(wave_scan(v, add_u64()), 63); }

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
    double f;       // log2 e / T
    int top_k;      // 0: no limit
    float top_p, min_p;
};

// the least weight that min_p, up to 1, keeps
__device__ __forceinline__ uint64_t least_weight(float min_p, uint64_t largest) {
    return min_p > 0.0f ? (uint64_t)ceil((double)min_p * (double)largest) : 0;
}

// the unit of the total that u names
__device__ __forceinline__ uint64_t draw_target(float u, uint64_t total) {
    const double at = u > 0.0f ? (double)u * (double)total : 0.0;
    return at >= (double)total ? total - 1 : min((uint64_t)at, total - 1);
}

// inclusive sums over the workgroup's threads; the same memory may be used
// again after the next barrier
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *s, uint64_t &all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v, add_u64());
    if (lane == 63) s[wave] = v;
    __syncthreads();
    const uint64_t t = row_scan(s[lane & (k_draw_waves - 1)], add_u64());
    all = read_lane(t, k_draw_waves - 1);
    return wave ? v + read_lane(t, wave - 1) : v;
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
    const bool sharp = !(fabsf(d0.xmax) < INFINITY) || !(d0.f < 1e300);
    const any_weigher any{(double)d0.xmax, d0.f};
    auto W = [&](float v) { return sharp ? (uint64_t)(v == d0.xmax) << k_w_sh : any(v); };
    const int top_k = d0.top_k;
    const float top_p = d0.top_p;
    // (the largest logit's own weight, which power() leaves 44 units below 2^40)
    const uint64_t wmin = least_weight(d0.min_p, W(d0.xmax));
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
                if (w < wmin) w = 0;
            }
            if (!draw) {
                run += w;
                continue;
            }
            const uint64_t inc = wave_scan(w, add_u64());
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
// for every pass, from L2 or the memory-side cache.
// - The largest logit; with top_k or top_p also one histogram over the distance
//   from it, of counts for top_k, of weights in 12 to 16 bits for top_p, which names the
//   bins that the border lies in.  In a long row both come from one pass: the
//   bins are counted from the largest of the first segments, with 22 binades
//   above it (a row that reaches beyond is counted again).
// - With a top_k the tokens down to that bin are put in order, which gives
//   top_p's and min_p's borders too, and the draw.
// - Otherwise the weights are summed by segment.  With a top_p the tokens of the
//   border's bins are collected meanwhile and their weights, from the exact sum
//   above them on, name the border exactly; if it is not among them (or
//   too many tokens are) the row takes draw_by_digits.
// - The segment that holds u's share is gone through again.
// Bound by a row's passes on one CU: one of loads, and one of weights (above).
// 256 rows of 131075: 22 us greedy (6 TB/s), 45 with a top_k, 52 without limits and
// 75 with a top_p (with an exact histogram of 64-bit weights for its border 106); by
// digits 606 with a top_k of 5000, 904 with a top_p too.
template <int R, bool MORE>
__global__ __launch_bounds__(k_draw_block) void k_draw(draw_args a) {
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // rows need no alignment
    __shared__ uint64_t s_list[k_list], s_sorted[k_list], s_order[k_list];
    __shared__ uint32_t s_place[k_list];
    __shared__ uint64_t s_seg[k_seg_max], s_scan[2][k_draw_waves];
    __shared__ uint64_t s_x;
    __shared__ int s_n, s_at, s_bin[4];
    __shared__ uint32_t s_cnt[4];
    uint32_t *const s_hist = reinterpret_cast<uint32_t *>(s_sorted);   // of counts
    static_assert(k_bins <= 2 * k_list, "");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n, segs = (n + k_seg - 1) / k_seg;
    const int64_t r = blockIdx.x;
    const float *x = a.logits + r * a.ld;

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
    auto kept = [&](auto f) {
#pragma unroll
        for (int i = 0; i < R; i++)
            if (i * k_draw_waves + wave < segs) f(i * k_draw_waves + wave, keep[i]);
    };
    auto each = [&](auto f) {
        float next[16];
        int seg = R * k_draw_waves + wave;
        if (MORE && seg < segs) load(seg, next);
        kept(f);
        if constexpr (MORE)
            for (; seg < segs; seg += k_draw_waves) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = next[e];
                if (seg + k_draw_waves < segs) load(seg + k_draw_waves, next);
                f(seg, v);
            }
    };

    const float T = uniform(a.temperature ? a.temperature[r] : 1.0f);
    draw_row D;
    D.f = uniform(1.4426950408889634 / (double)T);
    D.top_k = uniform(a.top_k ? a.top_k[r] : 0);
    if (D.top_k < 0 || D.top_k >= n) D.top_k = 0;
    D.top_p = uniform(a.top_p ? a.top_p[r] : 1.0f);
    if (!(D.top_p < 1.0f)) D.top_p = 1.0f;
    D.min_p = uniform(a.min_p ? a.min_p[r] : 0.0f);
    // (a min_p above 1 leaves the first token by rank, which is kept always)
    const bool greedy = !(T > 0.0f) || D.min_p > 1.0f;

    auto easy = [&]() -> bool {
        // Bins of a logit's distance from ref, which lies no more than k_head bins
        // below the largest logit; they never rise with the logit, and the last
        // holds all whose weight rounds to 0.
        const bool by_count = D.top_k > 0;
        const float scale = uniform((float)(k_bins_binade * D.f));
        const bool bins = !greedy && D.top_k <= k_small_k && (by_count || D.top_p < 1.0f) && scale < INFINITY;
        float ref = -INFINITY;
        auto place_of = [&](float v) {
            return __builtin_amdgcn_fmed3f(fmaf(ref - v, scale, (float)k_head), 0.0f, (float)(k_bins - 1));
        };
        auto bin_of = [&](float v) { return (int)place_of(v); };
        // By weight a token counts 2^shift at its bin's start and by the fraction of
        // its bin that it lies behind it less, as its weight does: a sum fits 32 bits,
        // and a bin's weight is known to half a unit, and 2^-18 for the third power's
        // term and the place's rounding.
        const int shift = by_count ? 0 : min(16, __clz(n));
        auto count_all = [&](const float *v) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int b = bin_of(v[e]);
                if (b < k_bins - 1) atomicAdd(&s_hist[b], 1u);
            }
        };
        auto weigh_all = [&](const float *v) {
            constexpr float step = 0.6931472f / k_bins_binade;
            const float unit = (float)(1 << shift);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float z = place_of(v[e]);
                const int b = (int)z;
                const float behind = z - (float)b;
                const float q = fmaf(fmaf(behind, 0.5f * step * step, -step) * behind, unit, unit);
                if (b < k_bins - 1) atomicAdd(&s_hist[b], (uint32_t)(q + 0.5f));
            }
        };
        auto block_max = [&](uint64_t v, uint64_t *s) {
            v = wave_scan(v, max_u64());
            if (lane == 63) s[wave] = v;
            __syncthreads();
            return read_lane(row_scan(s[lane & (k_draw_waves - 1)], max_u64()), k_draw_waves - 1);
        };

        // the largest logit, the first index that has it if that one is taken, and the bins
        float mx = -INFINITY;
        int at = 0x7fffffff;
        if (greedy) {
            each([&](int seg, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (v[e] > mx) {
                        mx = v[e];
                        at = index(seg, e);
                    }
            });
        } else if (bins && MORE) {
            // the bins in the same pass, from the largest of the segments in registers
            for (int i = tid; i < k_bins; i += k_draw_block) s_hist[i] = 0;
            kept([&](int, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, v[e]);
            });
            ref = key_value((uint32_t)block_max(order_key(mx), s_scan[1]));
            each([&](int, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, v[e]);
                if (by_count) count_all(v);
                else weigh_all(v);
            });
        } else {
            each([&](int, const float *v) {
#pragma unroll
                for (int e = 0; e < 16; e++) mx = fmaxf(mx, v[e]);
            });
        }
        const uint64_t best = block_max((uint64_t)order_key(mx) << 32 | (uint32_t)(0x7fffffff - at), s_scan[0]);
        const uint32_t kmax = (uint32_t)(best >> 32);
        if (kmax <= k_key_ninf || greedy) {
            if (tid == 0) {
                a.tokens[r] = kmax <= k_key_ninf ? -1 : 0x7fffffff - (int32_t)(uint32_t)best;
                if (a.probs) a.probs[r] = kmax <= k_key_ninf ? 0.0f : 1.0f;
            }
            return true;
        }
        D.xmax = key_value(kmax);
        if (D.top_k > k_small_k || !(fabsf(D.xmax) < INFINITY) || !(scale < INFINITY) || !weigher::fits(D.xmax, D.f))
            return false;
        const weigher W(D.xmax, D.f);
        const uint64_t wmin = uniform(least_weight(D.min_p, W(D.xmax)));

        // a token is kept if (key, index) does not come behind (bkey, bidx)
        uint32_t bkey = 0;
        int bidx = 0x7fffffff;
        bool bordered = false;
        if (bins) {
            if (!MORE || !((D.xmax - ref) * scale <= (float)k_head)) {   // (no bins yet, or not down to the largest)
                __syncthreads();
                for (int i = tid; i < k_bins; i += k_draw_block) s_hist[i] = 0;
                ref = D.xmax;
                __syncthreads();
                each([&](int, const float *v) {
                    if (by_count) count_all(v);
                    else weigh_all(v);
                });
            }
            if (tid == 0) s_n = 0;
            __syncthreads();
            uint32_t h[4];
            uint64_t sum = 0, counts;
#pragma unroll
            for (int i = 0; i < 4; i++) sum += h[i] = s_hist[tid * 4 + i];
            const uint32_t before_bin = (uint32_t)(block_scan(sum, s_scan[0], counts) - sum);
            if (tid < 4) s_bin[tid] = k_bins - 2, s_cnt[tid] = (uint32_t)counts;
            __syncthreads();
            // the first bin up to which v's sum (run: before the thread's) reaches
            // what is wanted, and the tokens before it (or, through, up to it)
            auto first_bin = [&](const uint64_t (&v)[4], uint64_t run, uint64_t want, int slot, bool through) {
                uint64_t next = run + v[0] + v[1] + v[2] + v[3];
                if (run >= want || next < want) return;
                uint32_t c = before_bin, at_b = 0;
                int b = 0;
#pragma unroll
                for (int i = 0; i < 3; i++)
                    if (b == i && run + v[i] < want) run += v[i], c += h[i], b++;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (b == i) at_b = h[i];
                s_bin[slot] = tid * 4 + b;
                s_cnt[slot] = through ? c + at_b : c;
            };
            int lo = 0, hi;   // the bins of the list
            bool cut = true;
            if (by_count) {
                // (fewer weigh anything: all bins but the last)
                const uint64_t v[4] = {h[0], h[1], h[2], h[3]};
                first_bin(v, before_bin, (uint64_t)D.top_k, 0, true);
                __syncthreads();
                hi = s_bin[0];
            } else {
                // the list: the bins in which the border may lie, by the estimates' errors
                // (of the sum up to it and of all, half a unit and 2^-18 each), or, where
                // those are many, those in which it does if errors mostly cancel
                uint64_t v[4], est = 0, all;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    est += v[i] = (uint64_t)((double)h[i] * (double)__builtin_amdgcn_exp2f(
                                      (float)(k_w_sh - shift) + (place_of(D.xmax) - (float)(tid * 4 + i)) * (1.0f / k_bins_binade)));
                const uint64_t run = block_scan(est, s_scan[1], all) - est;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const double p = (double)D.top_p * (double)all, off = (1.0 / (1 << shift) + 1.0 / 131072) / (i == 0 ? 1 : 16);
                    first_bin(v, run, (uint64_t)fmax(p * (1 - off), 1.0), 2 * i, false);
                    first_bin(v, run, min((uint64_t)fmax(p * (1 + off), 0.0) + 1, all), 2 * i + 1, true);
                }
                __syncthreads();
                const int of = s_cnt[1] - s_cnt[0] <= (uint32_t)(k_list - 64) << shift ? 0 : 2;
                lo = s_bin[of], hi = s_bin[of + 1];
                if (wmin) {
                    // min_p's border above top_p's: that one alone counts; at or below the
                    // list's first bin: what lies above the list is above it too
                    const int at = (int)(place_of(D.xmax) - log2f(D.min_p) * k_bins_binade);
                    cut = at + 1 >= s_bin[0];
                    lo = max(min(lo, at - 1), 0);
                }
            }
            if (cut) {
                auto push = [&](float v, int i) {
                    const int at = atomicAdd(&s_n, 1);
                    if (at < k_list) s_list[at] = (uint64_t)order_key(v) << 32 | (uint32_t)(0x7fffffff - i);
                };
                uint64_t all = 0, above = 0;
                asm volatile("" : "+v"(ref));   // bins are formed again, not kept in registers
                ref = uniform(ref);
                if (by_count) {
                    each([&](int seg, const float *v) {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (bin_of(v[e]) <= hi) push(v[e], index(seg, e));
                    });
                } else {
                    // the weights of all tokens, and by segment of those above the list
                    each([&](int seg, const float *v) {
                        uint64_t sum = 0;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const uint64_t w = W(v[e]);
                            const int b = bin_of(v[e]);
                            all += w;
                            sum += b < lo ? w : 0;
                            if (b >= lo && b <= hi) push(v[e], index(seg, e));
                        }
                        sum = wave_sum(sum);
                        above += sum;
                        if (lane == 0) s_seg[seg] = sum;
                    });
                    all = wave_sum(all);
                    if (lane == 0) s_scan[0][wave] = all, s_scan[1][wave] = above;
                }
                __syncthreads();
                const int m = s_n;
                if (m > k_list) return false;
                if (!by_count) {
                    all = above = 0;
                    for (int w = 0; w < k_draw_waves; w++) all += s_scan[0][w], above += s_scan[1][w];
                }
                if (by_count) {
                    order_items(s_list, s_sorted, s_place, m);
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
                    const bool in = tid < kept && w > 0 && w >= wmin;
                    if (tid < k_list / 2) s_list[tid] = 0;   // (what is not kept comes last)
                    __syncthreads();
                    // order by index: its complement above, its place in the ranking below
                    if (tid < kept) s_list[tid] = (uint64_t)(uint32_t)s_sorted[tid] << 32 | (in ? (uint32_t)tid + 1u : 0u);
                    __syncthreads();
                    uint64_t *const by_index = s_sorted + k_list / 2;   // (top_k <= k_list / 2)
                    order_items(s_list, by_index, s_place, kept);
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
                // top_p: the first of the list, as many as the weight still needs.  The
                // list's weights are summed over finer bins; the tokens of that in which
                // the border lies are put in order.
                const double p = ceil((double)D.top_p * (double)all);
                const uint64_t want = p >= 1.0 ? min((uint64_t)p, all) : 1;
                auto value = [&](uint64_t item) { return key_value((uint32_t)(item >> 32)); };
                const float fine = (float)k_draw_block / (float)(hi - lo + 1);
                auto fine_bin = [&](uint64_t item) {
                    return (int)fminf((place_of(value(item)) - (float)lo) * fine, (float)(k_draw_block - 1));
                };
                s_sorted[tid] = 0;
                if (tid == 0) s_at = -1, s_cnt[0] = 0;   // (s_n may still be read)
                __syncthreads();
                for (int i = tid; i < m; i += k_draw_block)
                    atomicAdd((unsigned long long *)&s_sorted[fine_bin(s_list[i])], (unsigned long long)W(value(s_list[i])));
                __syncthreads();
                uint64_t part;
                const uint64_t wf = s_sorted[tid], cf = above + block_scan(wf, s_scan[0], part);
                if (cf - wf < want && cf >= want) {
                    s_at = tid;
                    s_x = cf - wf;
                }
                __syncthreads();
                const int at = s_at;
                if (at < 0) return false;   // (the border is not in the list)
                uint64_t before = s_x;
                for (int i = tid; i < m; i += k_draw_block)
                    if (fine_bin(s_list[i]) == at) s_sorted[atomicAdd(&s_cnt[0], 1u)] = s_list[i];
                __syncthreads();
                const int few = (int)s_cnt[0];
                order_items(s_sorted, s_order, s_place, few);
                for (int i0 = 0; i0 < few; i0 += k_draw_block) {
                    const uint64_t w = i0 + tid < few ? W(value(s_order[i0 + tid])) : 0;
                    const uint64_t c = before + block_scan(w, s_scan[1 - (i0 / k_draw_block & 1)], part);
                    if (c - w < want && c >= want) s_at = i0 + tid;
                    before += part;
                }
                __syncthreads();
                const uint64_t item = s_order[s_at];
                for (int i = tid; i < m; i += k_draw_block) {
                    const uint64_t w = W(value(s_list[i]));
                    if (s_list[i] >= item && w >= wmin)
                        atomicAdd((unsigned long long *)&s_seg[(0x7fffffff - (int)(uint32_t)s_list[i]) / k_seg], (unsigned long long)w);
                }
                bkey = (uint32_t)(item >> 32);
                bidx = 0x7fffffff - (int)(uint32_t)item;
                bordered = true;
                __syncthreads();
            }
        }
        auto weigh = [&](float v, int i) {
            uint64_t w = W(v);
            if (w < wmin) w = 0;
            if (bordered) {
                const uint32_t k = order_key(v);
                if (k < bkey || (k == bkey && i > bidx)) w = 0;
            }
            return w;
        };
        if (!bordered) {
            auto sums = [&](auto keeps) {
                each([&](int seg, const float *v) {
                    uint64_t sum = 0;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint64_t w = W(v[e]);
                        sum += keeps(w) ? w : 0;
                    }
                    sum = wave_sum(sum);
                    if (lane == 0) s_seg[seg] = sum;
                });
            };
            if (wmin) sums([&](uint64_t w) { return w >= wmin; });
            else sums([](uint64_t) { return true; });
            __syncthreads();
        }
        uint64_t total;
        const uint64_t w = tid < segs ? s_seg[tid] : 0, c = block_scan(w, s_scan[0], total);
        const uint64_t target = draw_target(a.u[r], total);
        if (c > target && c - w <= target) {
            s_n = tid;
            s_x = target - (c - w);
        }
        __syncthreads();
        // the segment's tokens, one a thread
        const int i = s_n * k_seg + tid;
        const uint64_t left = s_x;
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
    if (!easy()) draw_by_digits(a, D, r, s_list, s_scan[0]);
}

}  // namespace lnship

using namespace lnship;

extern "C" {

int lnship_sample(const lnship_sample_args *a, void *stream) {
    if (!a) return fail(LNSHIP_EINVAL, "sample: null arguments%s");
    if (a->n_rows < 0 || a->n_vocab < 1) return fail(LNSHIP_EINVAL, "sample: bad shape%s");
    if (a->n_rows > 0x3fffff || a->n_vocab > k_draw_vocab) return fail(LNSHIP_ERANGE, "sample: too large%s");
    const int64_t ld = a->ld ? a->ld : a->n_vocab;
    if (ld < a->n_vocab) return fail(LNSHIP_EINVAL, "sample: bad shape%s");
    if (a->n_rows == 0) return 0;
    if (!a->logits || !a->u || !a->tokens) return fail(LNSHIP_EINVAL, "sample: null pointer%s");
    device_state *s = state();
    if (!s) return LNSHIP_ENOINIT;
    draw_args d{a->logits, ld, (int)a->n_vocab, a->temperature, a->top_k, a->top_p, a->min_p, a->u, a->tokens, a->probs};
    const dim3 grid((unsigned)a->n_rows), block(k_draw_block);
    hipStream_t st = (hipStream_t)stream;
    const int rounds = (int)((a->n_vocab + k_seg * k_draw_waves - 1) / (k_seg * k_draw_waves));
    // Up to two segments a wave stay in registers; of longer rows one, and the
    // others are read for each pass, which costs less than the registers' spills
    // (61 rows of 32000 logits 24.7 us in registers, 25.2 so; of 49152 31.2 so, 34.3 with
    // three in registers, one row 17.9 and 17.2; 256 of 131075 75.4 so, 76.9 with two).
    if (rounds == 1) hipLaunchKernelGGL((k_draw<1, false>), grid, block, 0, st, d);
    else if (rounds == 2) hipLaunchKernelGGL((k_draw<2, false>), grid, block, 0, st, d);
    else hipLaunchKernelGGL((k_draw<1, true>), grid, block, 0, st, d);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
