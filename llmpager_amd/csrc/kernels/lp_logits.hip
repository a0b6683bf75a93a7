// gfx950 kernels that read rows of logits: log probabilities of given tokens,
// the rows' entropies and their top alternatives.
//
// With M the row's largest logit, n the number of those equal to it, s = sum e^(x - M)
// over the others, S = n + s and Y = sum e^(x - M) (x - M):
//   log p(x) = (x - M) - log S,   entropy = log S - Y / S,   log S = log n + log(1 + s / n).
// Logits are read once.  A workgroup takes a part of a row and each of its
// waves 4096 bytes at a time, 16 logits a lane; M is the wave's running maximum,
// raised for the wave as a whole when a block passes it, which few blocks do.
// In a row that is sure of one token the entropy is all in what the other terms
// add to the 1 of the largest, so logits equal to M are counted apart and the
// others' sums kept beside the count to the end; sums of 16 are added up in 64 bits.
//
// The alternatives: lane i of a wave holds its i-th best as a key in the order of
// (value, lowest id first), and a block is looked through only if one of its
// logits reaches the last one that counts; of a block's own only those are taken
// that the lanes' two largest do not rule out.  Keys are put in one by one where
// they are few, else sorted 64 at a time across the lanes.
//
// A row's parts are joined by the workgroup that ends last.  777 rows of 151,936
// without alternatives take 91 us, 5.2 TB/s: a copy's rate.  32 rows of 151,936
// take 10 us without alternatives, 16 with one, 20 with twenty and 35 with 64; one
// such row 6 and 10 to 15: there the chain of a block's load, its exponentials,
// the sort and the join counts, 1 to 3 us each.
#include <type_traits>

#include "lp_rows.h"

using namespace lp;
using namespace lpk;

namespace {

constexpr int kPer = 16;               // logits of a lane in a block
constexpr int kBlock = 64 * kPer;      // and of a wave

__device__ __forceinline__ int wave_sum_i32(int v) {
    return (int)wave_reduce_u32((uint32_t)v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
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
            const float w = wave_top(mx);
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

// A logit as a whole number in the order of the alternatives: larger values
// first, lower ids first of equal ones (-0 and 0 are).  No number's is 0.
__device__ __forceinline__ uint32_t value_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The lane X further in the exclusive-or sense.
template <int X>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
    auto dpp = [](uint32_t u, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, decltype(ctrl)::value, 0xf, 0xf, false);
    };
    if constexpr (X == 1) return dpp(v, std::integral_constant<int, 0xb1>());
    if constexpr (X == 2) return dpp(v, std::integral_constant<int, 0x4e>());
    if constexpr (X == 3) return dpp(v, std::integral_constant<int, 0x1b>());
    if constexpr (X == 4) return xor_lane<7>(xor_lane<3>(v));
    if constexpr (X == 7) return dpp(v, std::integral_constant<int, 0x141>());   // mirrored within eight
    if constexpr (X == 8) return dpp(v, std::integral_constant<int, 0x128>());   // rotated within a row of 16
    if constexpr (X == 15) return dpp(v, std::integral_constant<int, 0x140>());  // mirrored within a row
    if constexpr (X == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return lane_id() & 16 ? r[0] : r[1];
    }
    if constexpr (X == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return lane_id() & 32 ? r[0] : r[1];
    }
    if constexpr (X == 31) return xor_lane<16>(xor_lane<15>(v));
    if constexpr (X == 63) return xor_lane<32>(xor_lane<31>(v));
}

// A key per lane: value key, then ~id; 0: none.
struct Keys {
    uint32_t hi = 0, lo = 0;

    // of each pair of lanes X apart the lower one keeps the larger key
    template <int X>
    __device__ __forceinline__ void order() {
        const uint32_t ph = xor_lane<X>(hi), pl = xor_lane<X>(lo);
        constexpr int bit = X >= 32 ? 32 : X >= 16 ? 16 : X >= 8 ? 8 : X >= 4 ? 4 : X >= 2 ? 2 : 1;
        const bool lower = (lane_id() & bit) == 0;
        const bool swap = (((uint64_t)ph << 32 | pl) > ((uint64_t)hi << 32 | lo)) == lower;
        hi = swap ? ph : hi;
        lo = swap ? pl : lo;
    }
    __device__ __forceinline__ void order_bitonic() {
        order<32>(), order<16>(), order<8>(), order<4>(), order<2>(), order<1>();
    }
    // largest first (a bitonic network whose halves are compared mirrored)
    __device__ __forceinline__ void sort() {
        order<1>();
        order<3>(), order<1>();
        order<7>(), order<2>(), order<1>();
        order<15>(), order<4>(), order<2>(), order<1>();
        order<31>(), order<8>(), order<4>(), order<2>(), order<1>();
        order<63>(), order<16>(), order<8>(), order<4>(), order<2>(), order<1>();
    }
    // the 64 largest of these and `k`, both sorted
    __device__ __forceinline__ void merge(const Keys& k) {
        const uint32_t ph = xor_lane<63>(k.hi), pl = xor_lane<63>(k.lo);
        const bool other = ((uint64_t)ph << 32 | pl) > ((uint64_t)hi << 32 | lo);
        hi = other ? ph : hi;
        lo = other ? pl : lo;
        order_bitonic();
    }
};

// The best logits a wave has seen, sorted.
struct Best : Keys {
    __device__ __forceinline__ void put(uint32_t h, uint32_t l) {  // one more, the same in all lanes
        const uint64_t x = (uint64_t)h << 32 | l;
        const int rank = __popcll(__ballot(((uint64_t)hi << 32 | lo) > x));
        const uint32_t ph = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, 0x138, 0xf, 0xf, false);  // the lane before
        const uint32_t pl = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, 0x138, 0xf, 0xf, false);
        const int lane = lane_id();
        hi = lane < rank ? hi : lane == rank ? h : ph;
        lo = lane < rank ? lo : lane == rank ? l : pl;
    }
    // A value key that at least `top` of the lanes' m1 and m2 reach: the largest
    // whose 12 last bits are zero.  What is below it is not among the best of
    // anything that holds those.
    static __device__ __forceinline__ uint32_t reached(uint32_t m1, uint32_t m2, int top) {
        uint32_t at = 0;
#pragma unroll
        for (int bit = 31; bit >= 12; --bit) {
            const uint32_t t = at | 1u << bit;
            at = (int)(__popcll(__ballot(m1 >= t)) + __popcll(__ballot(m2 >= t))) >= top ? t : at;
        }
        return at;
    }
    // Each lane's N keys (value keys h, 0: none).  A few are put in one by one
    // (about 170 cycles each); more go to a lane each through `room`, 64 keys of
    // LDS, and are sorted and merged (about 2,500 for up to 64 of them).
    template <int N, typename Lo>
    __device__ __forceinline__ void take(const uint32_t (&h)[N], const Lo& low, int top, volatile uint64_t* room) {
        uint32_t m1 = h[0], m2 = 0;
#pragma unroll
        for (int i = 1; i < N; ++i) m2 = max(m2, min(m1, h[i])), m1 = max(m1, h[i]);
        // none below the last that counts, nor below what the keys' own best are not
        uint32_t least = max(1u, (uint32_t)__builtin_amdgcn_readlane((int)hi, top - 1));
        if (__popcll(__ballot(m1 >= least)) > 8) least = max(least, reached(m1, m2, top));
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) count += __popcll(__ballot(h[i] >= least));
        if (count <= 12) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                for (uint64_t b = __ballot(h[i] >= least); b; b &= b - 1) {
                    const int l = __builtin_ctzll(b);
                    put((uint32_t)__builtin_amdgcn_readlane((int)h[i], l), (uint32_t)__builtin_amdgcn_readlane((int)low(i), l));
                }
            return;
        }
        int held = 0;
        auto flush = [&] {
            __builtin_amdgcn_wave_barrier();
            const int lane = lane_id();
            uint64_t key = 0;
            if (lane < held) key = room[lane];
            Keys k;
            k.hi = (uint32_t)(key >> 32), k.lo = (uint32_t)key;
            k.sort();
            if (__builtin_amdgcn_readfirstlane((int)hi))
                merge(k);
            else
                hi = k.hi, lo = k.lo;
            held = 0;
            __builtin_amdgcn_wave_barrier();
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t b = __ballot(h[i] >= least);
            const int n = __popcll(b);
            if (held + n > 64) flush();
            if (h[i] >= least)
                room[held + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0))] =
                    (uint64_t)h[i] << 32 | low(i);
            held += n;
        }
        flush();
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

// What a row's sums make of it: log(n + s), of a small r = s / n by the series of
// log(1 + r), whose first term left out is 2^-53 of it.
__device__ __forceinline__ double row_lse(const Sums& t) {
    if (t.m - t.m != 0.0f) return (double)__builtin_nanf("");
    const double n = (double)t.n, r = t.s / n;
    if (!(r < 0x1p-10)) return log(n + t.s);
    return (t.n == 1 ? 0.0 : log(n)) + r * (1.0 - r * (0.5 - r * (1.0 / 3.0 - r * (0.25 - r * 0.2))));
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
        const bool none = best.hi == 0;
        gptr_w<int>(a.ids)[at] = none ? -1 : (int)~best.lo;
        gptr_w<float>(a.top_logp)[at] = none ? __builtin_nanf("") : (float)((double)(key_value(best.hi) - t.m) - lse);
    }
}

// The sums of other waves or parts, one per lane (m = -inf, s = n = 0 where there
// is none), as one.
__device__ __forceinline__ Sums join(float m, double s, double y, int n) {
    Sums t;
    t.m = wave_top(m);
    if (m == -INFINITY) {
        s *= 0.0, y = 0.0, n = 0;  // -inf adds nothing; a NaN stays one
    } else if (m != t.m) {  // its maximum is one of the others
        const double f = (double)exp_neg(m - t.m), all = s + (double)n;
        y = f * (y + ((double)m - (double)t.m) * all);
        s = f * all, n = 0;
    }
    t.y = wave_sum_f64(y);
    t.s = wave_sum_f64(s);
    t.n = wave_sum_i32(n);
    return t;
}

// One part of a row by the whole workgroup, the result with its first wave.
template <bool TOP>
__device__ __forceinline__ void scan(const LogprobArgs& a, int row, int part, Sums& t, Best& best) {
    __shared__ float lm[4];
    __shared__ int ln[4];
    __shared__ double lsum[2][4];
    __shared__ uint64_t lk[TOP ? 4 : 1][64];  // a wave's room, then its best
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
    float last = -INFINITY;  // the last alternative that counts
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
            if (__ballot(mx >= last)) {
                uint32_t h[kPer];
                const int id0 = e + 4 * lane - skew;
                auto id = [&](int i) { return id0 + 256 * (i / 4) + i % 4; };
#pragma unroll
                for (int i = 0; i < kPer; ++i) h[i] = xs[i] == xs[i] && (uint32_t)id(i) < (uint32_t)n ? value_key(xs[i]) : 0u;
                best.take(h, [&](int i) { return ~(uint32_t)id(i); }, a.top, lk[wave]);
                const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)best.hi, a.top - 1);
                last = k ? key_value(k) : -INFINITY;
            }
        }
    }
    const double ws = wave_sum_f64(t.s), wy = wave_sum_f64(t.y);
    const int wn = wave_sum_i32(t.n);
    if (lane == 0) lm[wave] = t.m, lsum[0][wave] = ws, lsum[1][wave] = wy, ln[wave] = wn;
    if constexpr (TOP) lk[wave][lane] = (uint64_t)best.hi << 32 | best.lo;
    __syncthreads();
    if (wave) return;
    t = join(lane < 4 ? lm[lane & 3] : -INFINITY, lane < 4 ? lsum[0][lane & 3] : 0.0, lane < 4 ? lsum[1][lane & 3] : 0.0,
             lane < 4 ? ln[lane & 3] : 0);
    if constexpr (TOP)
        for (int w = 1; w < 4; ++w) {
            Keys k;
            k.hi = (uint32_t)(lk[w][lane] >> 32), k.lo = (uint32_t)lk[w][lane];
            best.merge(k);
        }
}

// Records: per (row, part) s, y, m and n (32 bytes); behind all of them the keys of its
// alternatives, a row's parts' one behind the other.
__device__ __forceinline__ uint64_t rec_at(const LogprobArgs& a, int row, int part) {
    return a.part + ((uint64_t)(uint32_t)row * (uint32_t)a.parts + (uint32_t)part) * 32;
}
__device__ __forceinline__ uint64_t keys_at(const LogprobArgs& a, int row, int part) {
    return rec_at(a, a.rows, 0) + ((uint64_t)(uint32_t)row * (uint32_t)a.parts + (uint32_t)part) * (uint32_t)(8 * a.top);
}
__device__ __forceinline__ void put64(uint64_t at, uint64_t v) { agent_store(reinterpret_cast<uint64_t*>(at), v); }
__device__ __forceinline__ uint64_t get64(uint64_t at) { return agent_load(reinterpret_cast<const uint64_t*>(at)); }

// The parts of a row joined by one wave: a part's sums per lane, the
// alternatives' keys 16 a lane.
template <bool TOP>
__device__ __forceinline__ void join_row(const LogprobArgs& a, int row) {
    const int lane = lane_id();
    float m = -INFINITY;
    double s = 0.0, y = 0.0;
    int n = 0;
    if (lane < a.parts) {
        const uint64_t r = rec_at(a, row, lane);
        s = __builtin_bit_cast(double, get64(r)), y = __builtin_bit_cast(double, get64(r + 8));
        const uint64_t mn = get64(r + 16);
        m = __uint_as_float((uint32_t)mn), n = (int)(mn >> 32);
    }
    Best best;
    if constexpr (TOP) {
        __shared__ uint64_t room[64];
        const uint64_t keys = keys_at(a, row, 0);
        for (int i0 = 0; i0 < a.parts * a.top; i0 += 1024) {
            uint32_t h[16], l[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int k = i0 + 64 * i + lane;
                uint64_t key = 0;
                if (k < a.parts * a.top) key = get64(keys + 8 * k);
                h[i] = (uint32_t)(key >> 32), l[i] = (uint32_t)key;
            }
            best.take(h, [&](int i) { return l[i]; }, a.top, room);
        }
    }
    finish(a, row, join(m, s, y, n), best);
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
        put64(r, __builtin_bit_cast(uint64_t, t.s));
        put64(r + 8, __builtin_bit_cast(uint64_t, t.y));
        put64(r + 16, (uint64_t)(uint32_t)t.n << 32 | __float_as_uint(t.m));
    }
    if (TOP && lane_id() < a.top) put64(keys_at(a, row, part) + 8 * lane_id(), (uint64_t)best.hi << 32 | best.lo);
    // the row's last part joins them: nothing waits
    int* const count = reinterpret_cast<int*>(a.sync) + row * kPagedStride;
    __builtin_amdgcn_s_waitcnt(0);
    int o = 0;
    if (lane_id() == 0) {
        o = atomicAdd(count, 1);
        if (o == a.parts - 1) agent_store(count, 0);  // zero for the next launch
    }
    if (__builtin_amdgcn_readfirstlane(o) == a.parts - 1) join_row<TOP>(a, row);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_logprobs(const LogprobArgs a) { logprobs_body<false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_logprobs_top(const LogprobArgs a) { logprobs_body<true>(a); }

// Arrival counters that are not a stream's own, before the launch that counts.
extern "C" __global__ void __launch_bounds__(256) lp_clear_words(const ClearArgs a) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i < a.n) agent_store(reinterpret_cast<int*>(a.at) + i, 0);
}
