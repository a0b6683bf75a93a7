// gfx950 kernels that decide which drafted tokens stay, from the target's logits of their
// rows and given random numbers.
//
// At temperature T the target's probabilities of a row are p(x) = e^((x - M) / T) / S.
// Drafts that were chosen, without probabilities of their own: a row's token is drawn, the
// first whose p with those of all before it passes the row's number, and where a child
// of the row's node is that token the walk goes on there: the tokens have exactly the
// target's distribution whatever was drafted.  Drafts that were sampled, the children of a
// node from q: with R_0 = p, Z_0 = 1 the children are tried in turn, child c is accepted if
// u q(c) Z_j < R_j(c), else what is left is
//   R_{j+1} = max(R_j - Z_j q, 0) = max(p - (a_j + Z_j) q, 0),  Z_{j+1} = sum R_{j+1},
// a_0 = 0, a_{j+1} = a_j + Z_j: one number says what is left of a row.  Behind the last child
// the next token is drawn from R / Z.  At temperature 0 both go by the largest logit.
//
// A draw is where a running sum over the vocabulary passes a border, and a value of 1e-7
// of the whole is many tokens' there: exponentials are made to 2^-42 and all sums in 64
// bits, so that the token is that of the formula.  Vector fp64 runs at fp32's rate here.
//
// A wave takes blocks of 1024 logits and leaves a record of each, its largest logit and the sum
// of e^ relative to that, so nothing is rescaled on the way; the row's last workgroup
// to end joins the records, finds the block in which the border lies and reads that one
// again.  Nothing waits.
#include <type_traits>

#include "lp_rows.h"

namespace {

constexpr double kNone = -800.0;  // e^ of it is 0

// e^d for kNone <= d <= 0: d = k ln 2 + r, |r| <= ln 2 / 2, Taylor's series of e^r, whose
// first term left out is 2^-42.
__device__ __forceinline__ double exp_f64(double d) {
    const double k = rint(d * 1.4426950408889634);
    const double r = __builtin_fma(-k, 0.6931471805599453, d);
    auto by_r = [&](double y, double c) { return __builtin_fma(y, r, c); };
    double y = by_r(2.7557319223985888e-7, 2.7557319223985893e-6);  // 1 / 10!, 1 / 9!, ...
    y = by_r(y, 2.4801587301587302e-5);
    y = by_r(y, 1.9841269841269841e-4);
    y = by_r(y, 1.3888888888888889e-3);
    y = by_r(y, 8.3333333333333333e-3);
    y = by_r(y, 4.1666666666666667e-2);
    y = by_r(y, 0.16666666666666667);
    y = by_r(y, 0.5);
    y = by_r(y, 1.0);
    y = by_r(y, 1.0);
    return __builtin_amdgcn_ldexp(y, (int)k);
}
// (a NaN counts as none here; rows with one are found by their logits)
__device__ __forceinline__ double exp_over(float x, float m, double inv_t) {
    return exp_f64(fmax(((double)x - (double)m) * inv_t, kNone));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double add_from(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Inclusive sums over the lanes (wave_incl_scan in 64 bits).
__device__ __forceinline__ double scan_f64(double v) {
    v = add_from<0x118, 0xf>(add_from<0x114, 0xf>(add_from<0x112, 0xf>(add_from<0x111, 0xf>(v))));
    return add_from<0x143, 0xc>(add_from<0x142, 0xa>(v));
}
__device__ __forceinline__ double lane_f64(double v, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l));
}
__device__ __forceinline__ float lane_f32(float v, int l) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); }
__device__ __forceinline__ int wave_least(int v) {
    return (int)wave_reduce_u32((uint32_t)v, 0x7fffffffu, [](uint32_t a, uint32_t b) { return (uint32_t)min((int)a, (int)b); });
}

__device__ __forceinline__ void put64(uint64_t at, uint64_t v) { agent_store(reinterpret_cast<uint64_t*>(at), v); }
__device__ __forceinline__ uint64_t get64(uint64_t at) { return agent_load(reinterpret_cast<const uint64_t*>(at)); }
__device__ __forceinline__ double getf64(uint64_t at) { return __builtin_bit_cast(double, get64(at)); }

constexpr int kPer = kVerifyBlock / 64;  // values of a lane in a block: 4 j + u is the block's 256 j + 4 lane + u
constexpr int kBad = 0x7fffffff;

// A block of a row; past its end `none`.
__device__ __forceinline__ void load_block(float (&v)[kPer], uint64_t row, int block, int n, float none) {
    const LP_GLOBAL float* const x = gptr<float>(row);
    typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) {
        const int e = block * kVerifyBlock + 256 * j + 4 * lane_id();
        if (e + 4 <= n) {
            const f32x4_u w = *reinterpret_cast<const LP_GLOBAL f32x4_u*>(x + e);
#pragma unroll
            for (int u = 0; u < 4; ++u) v[4 * j + u] = w[u];
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) v[4 * j + u] = e + u < n ? x[e + u] : none;
        }
    }
}

// The place in the block where the sums of v, `before` what went before them, pass thr; at
// rounding's edge the last that adds to them, -1 where none does.
__device__ __forceinline__ int find_in_block(const double (&v)[kPer], double before, double thr) {
    int at = -1;
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) {
        const double t = (v[4 * j] + v[4 * j + 1]) + (v[4 * j + 2] + v[4 * j + 3]);
        const double incl = before + scan_f64(t);
        const uint64_t some = __ballot(t > 0.0), hit = __ballot(incl > thr && t > 0.0);
        if (some) {
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
            double c = incl - t;
            int u = -1;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (u >= 0 && c > thr) continue;  // found
                c += v[4 * j + k];
                if (v[4 * j + k] > 0.0) u = k;
            }
            at = 256 * j + 4 * l + __builtin_amdgcn_readlane(u, l);
        }
        if (hit) return at;
        before = lane_f64(incl, 63);
    }
    return at;
}

// Which of a row's blocks holds the border: their sums w (block lane + 64 i) in order, and
// `share` of the whole.  The border and what goes before the block are left in thr and
// before; -1 where nothing adds to the sums.
__device__ __forceinline__ int find_block(const double (&w)[kVerifyLane], double share, double& thr, double& before) {
    double incl[kVerifyLane], all = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyLane; ++i) incl[i] = all + scan_f64(w[i]), all = lane_f64(incl[i], 63);
    thr = share * all;
    int at = -1;
    before = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyLane; ++i) {
        const uint64_t some = __ballot(w[i] > 0.0), hit = __ballot(incl[i] > thr && w[i] > 0.0);
        if (!some) continue;
        const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
        at = 64 * i + l, before = lane_f64(incl[i] - w[i], l);
        if (hit) break;
    }
    return at;
}

struct Seq {
    int t0, n;     // first token, nodes
    float temp;    // 0: the largest logit
    double inv_t;
};
__device__ __forceinline__ Seq seq_of(const VerifyArgs& a, int b) {
    Seq s;
    s.t0 = gptr<int>(a.q_starts)[b];
    s.n = min(gptr<int>(a.q_starts)[b + 1] - s.t0, a.max_q);
    if (s.t0 < 0 || s.t0 > a.tokens - s.n) s.n = 0;  // starts that name no tokens
    const float t = a.temps ? gptr<float>(a.temps)[b] : 1.0f;
    s.temp = t > 0.0f ? t : 0.0f;
    s.inv_t = 1.0 / (double)s.temp;
    return s;
}

__device__ __forceinline__ uint64_t logits_row(const VerifyArgs& a, int t) { return a.logits + (uint64_t)(uint32_t)t * (uint32_t)a.stride * 4; }
__device__ __forceinline__ uint64_t probs_row(const VerifyArgs& a, int t) { return a.probs + (uint64_t)(uint32_t)t * (uint32_t)a.probs_stride * 4; }
__device__ __forceinline__ uint64_t record(const VerifyArgs& a, int slot, int block) {
    return a.part + ((uint64_t)(uint32_t)slot * (uint32_t)a.blocks + (uint32_t)block) * 16;
}

// The records of a part of row t (those of slot `slot`), by the whole workgroup: the block's
// sum (NaN: a logit is NaN or infinite), its largest logit, and the first id of that.
__device__ __forceinline__ void scan_part(const VerifyArgs& a, const Seq& s, int t, int slot, int part) {
    const int wave = (int)(threadIdx.x >> 6), end = min(a.blocks, (part + 1) * a.per_part);
    const uint64_t row = logits_row(a, t);
    float x[kPer], next[kPer];
    int blk = part * a.per_part + wave;
    if (blk < end) load_block(next, row, blk, a.vocab, -INFINITY);
    for (; blk < end; blk += 4) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = next[i];
        if (blk + 4 < end) load_block(next, row, blk + 4, a.vocab, -INFINITY);
        float mx = x[0];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) mx = fmaxf(mx, x[i]), bad |= !(x[i] < INFINITY);
        mx = wave_top(mx);
        double sum = 0.0;
        int id = kBad;
        if (s.temp > 0.0f) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) sum += exp_over(x[i], mx, s.inv_t);
            sum = wave_sum_f64(sum);
        } else {
#pragma unroll
            for (int i = kPer - 1; i >= 0; --i) id = x[i] == mx ? blk * kVerifyBlock + 256 * (i / 4) + 4 * lane_id() + i % 4 : id;
            id = wave_least(id);
        }
        if (__ballot(bad)) sum = __builtin_nan("");
        if (lane_id() == 0) {
            const uint64_t r = record(a, slot, blk);
            put64(r, __builtin_bit_cast(uint64_t, sum));
            put64(r + 8, (uint64_t)(uint32_t)id << 32 | __float_as_uint(mx));
        }
    }
}

// A row's records joined by a wave.
struct Row {
    float m;                // the largest logit
    double s;               // the sum relative to it, NaN for a row from which nothing can be drawn
    double w[kVerifyLane];  // the sums of blocks lane + 64 i
    int first;              // the first id of the largest logit
};
__device__ __forceinline__ Row join_row(const VerifyArgs& a, const Seq& s, int slot) {
    Row r;
    float m[kVerifyLane];
    int id[kVerifyLane];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVerifyLane; ++i) {
        const int blk = lane_id() + 64 * i;
        r.w[i] = 0.0, m[i] = -INFINITY, id[i] = kBad;
        if (64 * i < a.blocks && blk < a.blocks) {
            const uint64_t at = record(a, slot, blk), mi = get64(at + 8);
            r.w[i] = getf64(at), m[i] = __uint_as_float((uint32_t)mi), id[i] = (int)(mi >> 32);
        }
        mx = fmaxf(mx, m[i]);
    }
    r.m = wave_top(mx);
    r.s = 0.0, r.first = kBad;
#pragma unroll
    for (int i = 0; i < kVerifyLane; ++i) {
        if (64 * i >= a.blocks) continue;
        if (m[i] == r.m) r.first = min(r.first, id[i]);
        r.w[i] *= s.temp > 0.0f ? exp_over(m[i], r.m, s.inv_t) : 1.0;
        r.s += wave_sum_f64(r.w[i]);
    }
    r.first = wave_least(r.first);
    if (r.m == -INFINITY) r.s = __builtin_nan("");
    return r;
}

// The token of row t that number u draws, -1: none can be.
__device__ __forceinline__ int draw(const VerifyArgs& a, const Seq& s, int t, const Row& r, float u) {
    if (r.s != r.s) return -1;
    if (s.temp == 0.0f) return r.first;
    double thr, before;
    const int blk = find_block(r.w, (double)u, thr, before);
    if (blk < 0) return -1;
    float x[kPer];
    load_block(x, logits_row(a, t), blk, a.vocab, -INFINITY);
    double v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = exp_over(x[i], r.m, s.inv_t);
    const int at = find_in_block(v, before, thr);
    return at < 0 ? -1 : blk * kVerifyBlock + at;
}

// What is left of a row's block: max(p - taken q, 0).
__device__ __forceinline__ void left_block(const VerifyArgs& a, const Seq& s, int t, int blk, float m, double inv_s, double taken, double (&v)[kPer]) {
    float x[kPer], q[kPer];
    load_block(x, logits_row(a, t), blk, a.vocab, -INFINITY);
    load_block(q, probs_row(a, t), blk, a.vocab, 0.0f);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = fmax(__builtin_fma(-taken, (double)q[i], exp_over(x[i], m, s.inv_t) * inv_s), 0.0);
}

// A counter's last arrival (the calling wave's stores are done before it counts).
__device__ __forceinline__ bool last_of(const VerifyArgs& a, int counter, int count) {
    int* const at = reinterpret_cast<int*>(a.sync) + (uint64_t)(uint32_t)counter * kPagedStride;
    __builtin_amdgcn_s_waitcnt(0);
    int o = 0;
    if (lane_id() == 0) {
        o = atomicAdd(at, 1);
        if (o == count - 1) agent_store(at, 0);  // zero for the next launch
    }
    return __builtin_amdgcn_readfirstlane(o) == count - 1;
}

__device__ __forceinline__ void put_node(const VerifyArgs& a, int b, int at, int node) {
    if (lane_id() == 0) gptr_w<int>(a.path)[(uint64_t)(uint32_t)b * (uint32_t)(a.max_depth + 1) + (uint32_t)at] = node;
}
// The walk's end after `len` nodes.
__device__ __forceinline__ void put_end(const VerifyArgs& a, int b, int len, int next) {
    for (int i = len + lane_id(); i <= a.max_depth; i += 64)
        gptr_w<int>(a.path)[(uint64_t)(uint32_t)b * (uint32_t)(a.max_depth + 1) + (uint32_t)i] = -1;
    if (lane_id() == 0) gptr_w<int>(a.kept)[b] = len, gptr_w<int>(a.next)[b] = next;
}

// Row t's statistics for the walk: its sum, {largest logit, draw}.
struct Stat {
    double s;
    float m;
    int z;
};
__device__ __forceinline__ void put_stat(const VerifyArgs& a, int t, const Row& r, int z) {
    if (lane_id()) return;
    const uint64_t at = a.stats + (uint64_t)(uint32_t)t * 16;
    put64(at, __builtin_bit_cast(uint64_t, r.s));
    put64(at + 8, (uint64_t)(uint32_t)z << 32 | __float_as_uint(r.m));
}
__device__ __forceinline__ Stat get_stat(const VerifyArgs& a, int t) {
    const uint64_t at = a.stats + (uint64_t)(uint32_t)t * 16, u = get64(at + 8);
    return Stat{getf64(at), __uint_as_float((uint32_t)u), (int)(u >> 32)};
}

// 64 nodes of a tree, one a lane: what each one's parent row says of it.
struct Nodes {
    int i0 = -1;          // the first one, -1: none are here
    int up, token;        // the parent (-2: none), the drafted token
    Stat own;             // of its own row
    bool fits;            // chosen drafts: it is the parent's draw; sampled ones: accepted as first child
    __device__ __forceinline__ void load(const VerifyArgs& a, const Seq& s, int first) {
        if (i0 == first) return;
        i0 = first;
        const int i = first + lane_id();
        up = -2, token = -1, fits = false, own = Stat{0.0, 0.0f, -1};
        if (i >= s.n) return;
        const int p = gptr<int>(a.parents)[s.t0 + i];
        token = gptr<int>(a.drafts)[s.t0 + i];
        own = get_stat(a, s.t0 + i);
        if (p < 0 || p >= i) return;
        up = p;
        const Stat st = get_stat(a, s.t0 + p);
        if ((uint32_t)token >= (uint32_t)a.vocab) return;
        if (a.probs && s.temp > 0.0f) {
            const float x = gptr<float>(logits_row(a, s.t0 + p))[token], q = gptr<float>(probs_row(a, s.t0 + p))[token];
            const float u = gptr<float>(a.uniforms)[s.t0 + i];
            fits = (double)u * (double)q < exp_over(x, st.m, s.inv_t) / st.s;
        } else {
            fits = token == st.z;
        }
    }
};

// A sequence's walk, by one wave, from node st.cur on until its end (true) or until what is
// left of a row has to be summed (false; then, with the blocks' sums in `sums`, the walk goes on).
__device__ __forceinline__ bool walk(const VerifyArgs& a, const Seq& s, int b, VerifyState& st, const double* sums) {
    const bool sampled = a.probs && s.temp > 0.0f;
    if (!(st.left > 0.0)) st.taken = 0.0, st.left = 1.0;  // nothing is left: p again
    Nodes N;
    for (;;) {
        N.load(a, s, st.cur & ~63);
        const int l = st.cur & 63;
        const double S = lane_f64(N.own.s, l);
        const float m = lane_f32(N.own.m, l);
        const int z = __builtin_amdgcn_readlane(N.own.z, l);
        if (S != S) {  // nothing can be drawn here
            put_end(a, b, st.len, -1);
            return true;
        }
        int to = -1;
        if (st.len <= a.max_depth)
            for (int i0 = max(st.cur, st.last) & ~63; i0 < s.n && to < 0; i0 += 64) {
                N.load(a, s, i0);
                uint64_t kids = __ballot(N.up == st.cur && i0 + lane_id() > st.last);
                if (!sampled || st.taken == 0.0) {
                    const uint64_t fit = kids & __ballot(N.fits);
                    if (!sampled) {
                        if (fit) to = i0 + __builtin_ctzll(fit);
                        continue;
                    }
                    // the first child is accepted or turned down
                    kids &= __ballot((uint32_t)N.token < (uint32_t)a.vocab);
                    if (!kids) continue;
                    const int k = __builtin_ctzll(kids);
                    if (fit >> k & 1) {
                        to = i0 + k;
                        continue;
                    }
                    st.last = i0 + k, st.taken = 1.0, st.pending = 1;
                    return false;
                }
                kids &= __ballot((uint32_t)N.token < (uint32_t)a.vocab);
                if (!kids) continue;
                const int k = __builtin_ctzll(kids), d = __builtin_amdgcn_readlane(N.token, k), t = s.t0 + st.cur;
                const double q = (double)gptr<float>(probs_row(a, t))[d], u = (double)gptr<float>(a.uniforms)[s.t0 + i0 + k];
                const double p = exp_over(gptr<float>(logits_row(a, t))[d], m, s.inv_t) / S;
                if (u * q * st.left < fmax(__builtin_fma(-st.taken, q, p), 0.0)) {
                    to = i0 + k;
                    continue;
                }
                st.last = i0 + k, st.taken += st.left, st.pending = 1;
                return false;
            }
        if (to >= 0) {
            st = VerifyState{to, to, st.len + 1, 0, 0.0, 1.0};
            put_node(a, b, st.len - 1, to);
            continue;
        }
        int next = z;
        if (sampled) {
            const int t = s.t0 + st.cur;
            const float u = gptr<float>(a.uniforms)[s.t0];
            if (st.taken == 0.0) {
                next = draw(a, s, t, join_row(a, s, t), u);
            } else {
                double w[kVerifyLane], thr, before, v[kPer];
#pragma unroll
                for (int i = 0; i < kVerifyLane; ++i) w[i] = lane_id() + 64 * i < a.blocks ? sums[lane_id() + 64 * i] : 0.0;
                const int blk = find_block(w, (double)u, thr, before);
                left_block(a, s, t, max(blk, 0), m, 1.0 / S, st.taken, v);
                next = max(blk, 0) * kVerifyBlock + max(find_in_block(v, before, thr), 0);
            }
        }
        put_end(a, b, st.len, next);
        return true;
    }
}

}  // namespace

// The sequence of row t, batch where it has none: also where the starts do not rise, so that
// no workgroup of the launch counts itself then.
__device__ __forceinline__ int sequence_of_row(const VerifyArgs& a, int t) {
    int b = 0;
    bool falls = false;
    for (int i = 0; i < a.batch; i += 64) {
        const int at = i + lane_id();
        bool past = false;
        if (at < a.batch) {
            const int from = gptr<int>(a.q_starts)[at], to = gptr<int>(a.q_starts)[at + 1];
            past = to <= t, falls |= to < from;
        }
        b += __popcll(__ballot(past));
    }
    return __ballot(falls) ? a.batch : __builtin_amdgcn_readfirstlane(b);
}

// Every row at once: workgroup (row, part).  A row's last workgroup joins its records, a
// sequence's last row walks down its tree.
extern "C" __global__ void __launch_bounds__(256) lp_verify_rows(const VerifyArgs a) {
    const int t = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - t * a.parts, wave = (int)(threadIdx.x >> 6);
    if (blockIdx.x == 0 && wave == 3)  // sequences without a token
        for (int b = lane_id(); b < a.batch; b += 64) {
            if (seq_of(a, b).n > 0) continue;
            for (int i = 0; i <= a.max_depth; ++i) gptr_w<int>(a.path)[(uint64_t)(uint32_t)b * (uint32_t)(a.max_depth + 1) + (uint32_t)i] = -1;
            gptr_w<int>(a.kept)[b] = 0, gptr_w<int>(a.next)[b] = -1;
            if (a.probs) gptr_w<VerifyState>(a.state)[b].pending = 0;
        }
    const int b = sequence_of_row(a, t);
    if (b >= a.batch) return;  // whole workgroups, here and below
    const Seq s = seq_of(a, b);
    if (t < s.t0 || t - s.t0 >= s.n) return;
    scan_part(a, s, t, t, part);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (wave) return;
    if (a.parts > 1 && !last_of(a, t, a.parts)) return;
    const Row r = join_row(a, s, t);
    const bool sampled = a.probs && s.temp > 0.0f;
    put_stat(a, t, r, sampled ? -1 : draw(a, s, t, r, gptr<float>(a.uniforms)[t]));
    if (!last_of(a, a.row_counters + b, s.n)) return;
    VerifyState st{0, 0, 1, 0, 0.0, 1.0};
    put_node(a, b, 0, 0);
    walk(a, s, b, st, nullptr);
    if (a.probs && lane_id() == 0) gptr_w<VerifyState>(a.state)[b] = st;
}

// What is left of a row, for the sequences whose walk stands there: workgroup (sequence,
// part) sums a wave's blocks, the last one goes on with the walk, and where that needs
// another row's or more taken from this one, sums that alone.
extern "C" __global__ void __launch_bounds__(64 * kVerifyWaves) lp_verify_left(const VerifyArgs a) {
    __shared__ double sums[64 * kVerifyLane];
    __shared__ VerifyState now;
    __shared__ int flag;
    const int b = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - b * a.parts;
    const int wave = (int)(threadIdx.x >> 6), lane = lane_id();
    VerifyState st = gptr<VerifyState>(a.state)[b];
    if (!st.pending) return;  // whole workgroups, here and below
    const Seq s = seq_of(a, b);
    const uint64_t mine = a.left + (uint64_t)(uint32_t)b * (uint32_t)a.blocks * 8;
    auto sum_block = [&](int blk) {
        const Stat r = get_stat(a, s.t0 + st.cur);
        double v[kPer], sum = 0.0;
        left_block(a, s, s.t0 + st.cur, blk, r.m, 1.0 / r.s, st.taken, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += v[i];
        return wave_sum_f64(sum);
    };
    for (int blk = part * a.per_part + wave; blk < min(a.blocks, (part + 1) * a.per_part); blk += kVerifyWaves) {
        const double sum = sum_block(blk);
        if (lane == 0) put64(mine + 8 * blk, __builtin_bit_cast(uint64_t, sum));
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (wave == 0) {
        const bool last = a.parts == 1 || last_of(a, a.row_counters + b, a.parts);
        if (lane == 0) flag = last;
    }
    __syncthreads();
    if (!flag) return;
    for (int i = threadIdx.x; i < a.blocks; i += 64 * kVerifyWaves) sums[i] = getf64(mine + 8 * i);
    for (;;) {
        __syncthreads();
        if (wave == 0) {
            double z = 0.0;
            for (int i = lane; i < a.blocks; i += 64) z += sums[i];
            st.left = wave_sum_f64(z), st.pending = 0;
            const bool done = walk(a, s, b, st, sums);
            if (lane == 0) now = st, flag = done;
        }
        __syncthreads();
        if (flag) return;
        st = now;
        for (int blk = wave; blk < a.blocks; blk += kVerifyWaves) {
            const double sum = sum_block(blk);
            if (lane == 0) sums[blk] = sum;
        }
    }
}

// By levels, chosen drafts: workgroup (sequence, part) of the row that the walk stands at,
// whose last one goes a node down, for the next launch.
extern "C" __global__ void __launch_bounds__(256) lp_verify_level(const VerifyArgs a) {
    const int b = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - b * a.parts, wave = (int)(threadIdx.x >> 6);
    const Seq s = seq_of(a, b);
    const int cur = a.level ? gptr<int>(a.state)[b] : 0;
    if (s.n <= 0) {
        if (a.level == 0 && part == 0 && wave == 0) {
            put_end(a, b, 0, -1);
            if (lane_id() == 0) gptr_w<int>(a.state)[b] = -1;
        }
        return;
    }
    if (cur < 0) return;  // whole workgroups
    const int t = s.t0 + cur;
    scan_part(a, s, t, b, part);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (wave) return;
    if (a.parts > 1 && !last_of(a, a.row_counters + b, a.parts)) return;
    const int z = draw(a, s, t, join_row(a, s, b), gptr<float>(a.uniforms)[t]);
    int to = -1;
    if (z >= 0 && a.level < a.max_depth)
        for (int i0 = cur & ~63; i0 < s.n && to < 0; i0 += 64) {
            const int i = i0 + lane_id();
            const bool fits = i < s.n && i > cur && gptr<int>(a.parents)[s.t0 + i] == cur && gptr<int>(a.drafts)[s.t0 + i] == z;
            const uint64_t fit = __ballot(fits);
            if (fit) to = i0 + __builtin_ctzll(fit);
        }
    put_node(a, b, a.level, cur);
    if (to < 0) put_end(a, b, a.level + 1, z);
    if (lane_id() == 0) gptr_w<int>(a.state)[b] = to;
}
