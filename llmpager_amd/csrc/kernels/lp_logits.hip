// gfx950 kernels that read rows of logits: log probabilities of given tokens,
// the rows' entropies and their top alternatives.
//
// With M the row's largest logit, S = sum e^(x - M) and Y = sum e^(x - M) (x - M):
//   log p(x) = (x - M) - log S,   entropy = log S - Y / S.
// Logits are read once.  A workgroup takes a part of a row and each of its
// waves 4096 bytes at a time, 16 logits a lane; M is the wave's running maximum,
// raised for the wave as a whole when a block passes it, which few blocks do.
// In a row that is sure of one token the entropy is all in what the other terms
// add to the 1 of the largest, so logits equal to M are counted apart and the
// others' sums kept beside the count; sums of 16 are added up in 64 bits.
//
// The alternatives: lane i of a wave holds its i-th best (value, id), and a
// block is looked through only if one of its logits reaches the last one that
// counts.  In rows of independent logits a wave of n takes about top (1 +
// ln(n / top)) of them, one exchange between neighbouring lanes each.
#include "lp_device.h"

using namespace lp;
using namespace lpk;

namespace {

constexpr int kPer = 16;               // logits of a lane in a block
constexpr int kBlock = 64 * kPer;      // and of a wave

__device__ __forceinline__ double wave_sum_f64(double v) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// e^d for d <= 0: the hardware's base-2 exponential, with what the product
// d log2 e is rounded by put back, so that it is good to a few units of 2^-24
// at any d.
__device__ __forceinline__ float exp_neg(float d) {
    constexpr float L = 1.44269504088896341f, LO = 1.925963033500e-8f;
    const float t = d * L;
    const float r = __builtin_fmaf(d, LO, __builtin_fmaf(d, L, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    // -inf leaves r without meaning: e is 0 there
    return d < -150.0f ? e : __builtin_fmaf(e * r, 0.69314718055994531f, e);
}

// The running maximum and sums of a wave's logits; s and y are the lane's.
struct Sums {
    float m = -INFINITY;
    double s = 0.0, y = 0.0;  // of logits below m
    int n = 0;                // logits equal to m

    // to a larger maximum
    __device__ __forceinline__ void raise(float to) {
        const double all = s + (double)n;
        if (m == -INFINITY) {
            s = all * 0.0, y = 0.0;  // -inf adds nothing; a NaN stays one
        } else {
            const double f = (double)exp_neg(m - to);
            y = f * (y + ((double)m - (double)to) * all);
            s = f * all;
        }
        n = 0;
        m = to;
    }
    __device__ __forceinline__ void add(const float (&x)[kPer], float mx) {
        if (__ballot(mx >= m)) {
            const float w = wave_max(mx);
            if (w > m) raise(w);
            float bs = 0.0f, by = 0.0f;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const bool top = x[i] == m;
                const float d = x[i] - m, e = top ? 0.0f : exp_neg(d);
                n += top;
                bs += e;
                by = __builtin_fmaf(e, top ? 0.0f : fmaxf(d, -200.0f), by);
            }
            s += (double)bs, y += (double)by;
            return;
        }
        float bs = 0.0f, by = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float d = x[i] - m, e = exp_neg(d);
            bs += e;
            by = __builtin_fmaf(e, fmaxf(d, -200.0f), by);  // 0 for -inf; NaN through e
        }
        s += (double)bs, y += (double)by;
    }
};

// The best (value, id) pairs a wave has seen, lane i the i-th: larger values
// first, lower ids first of equal ones.  NaN enters nowhere.
struct Best {
    float v = -INFINITY;
    int id = INT32_MAX;
    float tv = -INFINITY;  // the last that counts
    int tid = INT32_MAX;

    __device__ __forceinline__ void put(float x, int i, int top) {  // x, i the same in all lanes
        const bool before = v > x || (v == x && id < i);
        const int rank = __popcll(__ballot(before));
        const float pv = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x138, 0xf, 0xf, false));
        const int pi = __builtin_amdgcn_update_dpp(0, id, 0x138, 0xf, 0xf, false);  // the lane before
        const int lane = lane_id();
        v = lane < rank ? v : lane == rank ? x : pv;
        id = lane < rank ? id : lane == rank ? i : pi;
        tv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), top - 1));
        tid = __builtin_amdgcn_readlane(id, top - 1);
    }
    // A value that at least `top` lanes' mx reach: the largest whose 12 last
    // bits, in the order of their bit patterns, are zero.  What is below it is
    // not among the best of anything that holds those mx.
    static __device__ __forceinline__ float reached(float mx, int top) {
        const uint32_t b = __float_as_uint(mx), key = b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
        uint32_t at = 0;
#pragma unroll
        for (int bit = 31; bit >= 12; --bit) {
            const uint32_t t = at | 1u << bit;
            at = __popcll(__ballot(key >= t)) >= top ? t : at;
        }
        // (the patterns below -inf's are NaNs)
        return fmaxf(at & 0x80000000u ? __uint_as_float(at ^ 0x80000000u) : __uint_as_float(~at), -INFINITY);
    }
    // each lane's (x, i) where `on`
    __device__ __forceinline__ void take(float x, int i, bool on, int top) {
        uint64_t left = ~0ull;
        for (;;) {
            const uint64_t b = __ballot(on && (x > tv || (x == tv && i < tid))) & left;
            if (!b) return;
            const int l = __builtin_ctzll(b);
            left &= ~(1ull << l);
            put(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)), __builtin_amdgcn_readlane(i, l), top);
        }
    }
};

// Four logits from index e of a row; those outside [0, n) are -inf.
__device__ __forceinline__ f32x4_t load4(const LP_GLOBAL float* x, int e, int n) {
    if (e >= 0 && e + 4 <= n) return *reinterpret_cast<const LP_GLOBAL f32x4_t*>(x + e);
    f32x4_t r;
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = e + u >= 0 && e + u < n ? x[e + u] : -INFINITY;
    return r;
}

// What a row's sums make of it.
__device__ __forceinline__ double row_lse(const Sums& t) {
    return t.m - t.m == 0.0f ? log(t.s + (double)t.n) : (double)__builtin_nanf("");
}

// The row's results, by the wave that holds its sums and best: lane i alternative i.
__device__ __forceinline__ void finish(const LogprobArgs& a, int row, const Sums& t, const Best& best) {
    const double lse = row_lse(t);
    const LP_GLOBAL float* x = gptr<float>(a.logits + (uint64_t)row * (uint32_t)a.stride * 4);
    const int lane = lane_id();
    if (lane == 0) {
        if (a.targets) {
            const int k = gptr<int>(a.targets)[row];
            gptr_w<float>(a.logp)[row] = (uint32_t)k < (uint32_t)a.vocab ? (float)((double)(x[k] - t.m) - lse) : 0.0f;
        }
        if (a.entropy) gptr_w<float>(a.entropy)[row] = (float)(lse - t.y / (t.s + (double)t.n));
    }
    if (lane < a.top) {
        const uint64_t at = (uint64_t)row * (uint32_t)a.top + (uint32_t)lane;
        const bool none = best.id == INT32_MAX;
        gptr_w<int>(a.ids)[at] = none ? -1 : best.id;
        gptr_w<float>(a.top_logp)[at] = none ? __builtin_nanf("") : (float)((double)(best.v - t.m) - lse);
    }
}

// The sums of other waves or parts, one per lane (m = -inf, s = 0 where there
// is none), as one.
__device__ __forceinline__ Sums join(float m, double s, double y) {
    Sums t;
    t.m = wave_max(m);
    double f = m == t.m ? 1.0 : (double)exp_neg(m - t.m);
    if (m == -INFINITY) {
        f = 0.0;
        y = 0.0, m = t.m;
    }
    // s holds the count of its maximum
    t.y = wave_sum_f64(f * (y + (m == t.m ? 0.0 : ((double)m - (double)t.m) * s)));
    t.s = wave_sum_f64(f * s);
    return t;
}

// One part of a row by the whole workgroup, the result with its first wave.
template <bool TOP>
__device__ __forceinline__ void scan(const LogprobArgs& a, int row, int part, Sums& t, Best& best) {
    __shared__ float lm[4];
    __shared__ double lsum[2][4];
    __shared__ float lv[TOP ? 4 : 1][64];
    __shared__ int li[TOP ? 4 : 1][64];
    const uint64_t at = a.logits + (uint64_t)row * (uint32_t)a.stride * 4;
    const LP_GLOBAL float* x = gptr<float>(at);
    const int wave = (int)(threadIdx.x >> 6), lane = lane_id();
    // 16-byte pieces from the address at or before the row's first
    const int skew = (int)(at >> 2 & 3), n = a.vocab;
    const int e0 = part * a.per_part, e1 = min(n + skew, e0 + a.per_part);
    f32x4_t v[4];
    auto load = [&](int e) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = load4(x, e + 4 * (lane + 64 * j) - skew, n);
    };
    int e = e0 + wave * kBlock;
    if (e < e1) load(e);
    for (; e < e1; e += 4 * kBlock) {
        float xs[kPer];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < 4; ++u) xs[4 * j + u] = v[j][u];
        if (e + 4 * kBlock < e1) load(e + 4 * kBlock);
        float mx = xs[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) mx = fmaxf(mx, xs[i]);
        t.add(xs, mx);
        if constexpr (TOP) {
            const uint64_t b = __ballot(mx >= best.tv);
            if (b) {
                // many: first what the block's own best are not below
                const float least = __popcll(b) > 8 ? Best::reached(mx, a.top) : -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int id = e + 4 * (lane + 64 * j) - skew + u;
                        best.take(xs[4 * j + u], id, xs[4 * j + u] >= least && id >= 0 && id < n, a.top);
                    }
            }
        }
    }
    const double ws = wave_sum_f64(t.s + (double)t.n), wy = wave_sum_f64(t.y);
    if (lane == 0) lm[wave] = t.m, lsum[0][wave] = ws, lsum[1][wave] = wy;
    if constexpr (TOP) lv[wave][lane] = best.v, li[wave][lane] = best.id;
    __syncthreads();
    if (wave) return;
    t = join(lane < 4 ? lm[lane & 3] : -INFINITY, lane < 4 ? lsum[0][lane & 3] : 0.0, lane < 4 ? lsum[1][lane & 3] : 0.0);
    if constexpr (TOP)
        for (int w = 1; w < 4; ++w) best.take(lv[w][lane], li[w][lane], lane < a.top && li[w][lane] != INT32_MAX, a.top);
}

// Records: per (row, part) s, y, m (32 bytes), then its alternatives.
__device__ __forceinline__ uint64_t rec_at(const LogprobArgs& a, int row, int part) {
    return a.part + ((uint64_t)(uint32_t)row * (uint32_t)a.parts + (uint32_t)part) * (uint32_t)logprob_rec(a.top);
}

template <bool TOP>
__device__ __forceinline__ void logprobs_body(const LogprobArgs& a) {
    const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x % a.parts;
    Sums t;
    Best best;
    scan<TOP>(a, row, part, t, best);
    if (threadIdx.x >= 64) return;
    if (a.parts == 1) {
        finish(a, row, t, best);
        return;
    }
    const uint64_t r = rec_at(a, row, part);
    if (lane_id() == 0) {
        gptr_w<double>(r)[0] = t.s;
        gptr_w<double>(r)[1] = t.y;
        gptr_w<float>(r)[4] = t.m;
    }
    if (TOP && lane_id() < a.top) {
        gptr_w<float>(r + 32)[lane_id()] = best.v;
        gptr_w<int>(r + 32 + 4 * a.top)[lane_id()] = best.id;
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_logprobs(const LogprobArgs a) { logprobs_body<false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_logprobs_top(const LogprobArgs a) { logprobs_body<true>(a); }

// The parts of a row joined: a workgroup per row, its first wave the sums (a
// part per lane), all four the alternatives.
extern "C" __global__ void __launch_bounds__(256) lp_logprobs_join(const LogprobArgs a) {
    __shared__ float lv[4][64];
    __shared__ int li[4][64];
    const int row = blockIdx.x, wave = (int)(threadIdx.x >> 6), lane = lane_id();
    Best best;
    if (a.top) {
        for (int p = wave; p < a.parts; p += 4) {
            const uint64_t r = rec_at(a, row, p) + 32;
            const bool on = lane < a.top;
            float v = 0.0f;
            int id = INT32_MAX;
            if (on) v = gptr<float>(r)[lane], id = gptr<int>(r + 4 * a.top)[lane];
            best.take(v, id, on && id != INT32_MAX, a.top);
        }
        lv[wave][lane] = best.v, li[wave][lane] = best.id;
        __syncthreads();
    }
    if (wave) return;
    float m = -INFINITY;
    double s = 0.0, y = 0.0;
    if (lane < a.parts) {
        const uint64_t r = rec_at(a, row, lane);
        s = gptr<double>(r)[0], y = gptr<double>(r)[1], m = gptr<float>(r)[4];
    }
    const Sums t = join(m, s, y);
    if (a.top)
        for (int w = 1; w < 4; ++w) best.take(lv[w][lane], li[w][lane], lane < a.top && li[w][lane] != INT32_MAX, a.top);
    finish(a, row, t, best);
}
