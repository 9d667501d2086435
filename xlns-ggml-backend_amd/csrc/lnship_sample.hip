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
constexpr int64_t k_draw_vocab = (int64_t)1 << 22;   // their sum stays below 2^63

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

// The weight e^((x - x_max) / T) in units of 2^-40.  The exponent is formed in
// 64 bits (32 would lose what tells two sums apart), its fraction's power in
// 32: 24 bits of every weight.
struct weigher {
    double xmax, f;   // f = log2 e / T
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const double d = (double)x - xmax;
        const double y = x == (float)xmax ? 0.0 : d * f;
        if (!(y > -64.0)) return 0;
        const double n = rint(y);
        // 2^r in [2^-1/2, 2^1/2]: an integer in units of 2^-24
        const uint64_t q = (uint64_t)(uint32_t)(__builtin_amdgcn_exp2f((float)(y - n)) * 16777216.0f);
        const int sh = k_w_sh - 24 + (int)n;
        return sh >= 0 ? q << sh : q >> -sh;
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

// One workgroup a row.  The border of the top_k first, then that of top_p, is
// found digit by digit of the ordered keys, over a histogram of counts and
// weights of the keys that have the digits so far; ties at a border are kept
// from the lowest index on.
__global__ __launch_bounds__(k_draw_block) void k_draw(draw_args a) {
    __shared__ uint64_t s_w[256];
    __shared__ uint32_t s_c[256];
    __shared__ uint64_t s_u64[k_draw_waves];
    __shared__ uint32_t s_u32[k_draw_waves];
    __shared__ uint32_t s_digit;
    __shared__ uint64_t s_above_w;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
    const int64_t r = blockIdx.x;
    const float *x = a.logits + r * a.ld;

    // the largest key, and the first index that has it
    uint64_t best = 0;
    for (int i = tid; i < n; i += k_draw_block)
        best = max(best, (uint64_t)order_key(x[i]) << 32 | (uint32_t)(0x7fffffff - i));
    for (int d = 32; d; d >>= 1) best = max(best, (uint64_t)__shfl_xor(best, d));
    if (lane == 0) s_u64[wave] = best;
    __syncthreads();
    for (int w = 0; w < k_draw_waves; w++) best = max(best, s_u64[w]);
    __syncthreads();
    const uint32_t kmax = (uint32_t)(best >> 32);
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    if (kmax <= k_key_ninf || !(T > 0.0f)) {
        if (tid == 0) {
            a.tokens[r] = kmax <= k_key_ninf ? -1 : 0x7fffffff - (int32_t)(uint32_t)best;
            if (a.probs) a.probs[r] = kmax <= k_key_ninf ? 0.0f : 1.0f;
        }
        return;
    }
    const float xmax = key_value(kmax);
    const weigher W{(double)xmax, 1.4426950408889634 / (double)T};

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

    const int top_k = a.top_k ? a.top_k[r] : 0;
    if (top_k > 0 && top_k < n) {
        // (fewer logits above -inf than top_k: no border)
        uint64_t c = 0;
        for (int i = tid; i < n; i += k_draw_block) c += order_key(x[i]) > k_key_ninf;
        if (block_sum(c) > (uint64_t)top_k) select(true, (uint64_t)top_k);
    }
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
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
    // (the largest logit weighs 2^40 units)
    const float min_p = a.min_p ? a.min_p[r] : 0.0f;
    const double wmin = min_p > 0.0f ? fmin((double)min_p, 1.0) * (double)((uint64_t)1 << k_w_sh) : 0.0;

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
    const float u = a.u[r];
    const double at = u > 0.0f ? (double)u * (double)total : 0.0;
    const uint64_t target = at >= (double)total ? total - 1 : min((uint64_t)at, total - 1);
    pass(target, true, total);
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
    hipLaunchKernelGGL(k_draw, dim3((unsigned)a->n_rows), dim3(k_draw_block), 0, (hipStream_t)stream, d);
    LNSHIP_HIP(hipGetLastError());
    return 0;
}

}  // extern "C"
