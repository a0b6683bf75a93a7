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
// of the whole is many tokens' there: exponentials are made to 2^-40 and all sums in 64
// bits, so that the token is that of the formula.  Vector fp64 runs at fp32's rate here.
//
// A wave takes blocks of 1024 logits and leaves a record of each, its largest logit and the sum
// of e^ relative to that, so nothing is rescaled on the way; the row's last workgroup
// to end joins the records, finds the block in which the border lies and reads that one
// again.  Nothing waits for another workgroup, but that those of lp_verify_path look for the next
// node for a while (kLooks) and then leave.
#include <type_traits>

#include "lp_rows.h"

namespace {

// A token 660 or more below the row's largest can't be drawn: its e^, made from no lower exponent
// than kNone, is e^-660 at most (kNothing is 1e-11 of it above that, more than its error).  A sum
// of four or of a block's 1024 holds a larger weight than `least` if it is above that many times it,
// and some to spare at each step, so that what is found in the sums is found below them too.
constexpr double kNone = -700.0, kNothing = 2.3208225942028e-287;
constexpr double kOfFour = 4.1, kOfBlock = 1100.0;

// e^((x - m) / T): d = n ln 2 + r, |r| <= ln 2 / 2, and 2^n by the exponent's bits.  The
// polynomial has the smallest largest relative error of those of degree 8 that are 1 at
// 0: 2^-40.  (Taylor's of degree 10 with rounding and scaling instructions of their own is
// 22 fp64 instructions of 2.1 ns a wave and SIMD, this 17 and one of 1.3.)  N at a time, a
// step of all before the next, for a step waits for the one before it.
// (A NaN counts as none here; rows with one are found by their logits.)
template <int N>
__device__ __forceinline__ void exp_over(const float* x, float m, double inv_t, double* e) {
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: the sum's last bits are the whole number
    constexpr double C[8] = {0.00019914665993177232, 0.0013889154943716253, 0.008333268780697685, 0.04166666453742114,
                             0.16666666873210403, 0.500000000045801, 0.999999999983073, 1.0};
    double d[N], t[N], y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = ((double)x[i] - (double)m) * inv_t;
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = fmax(d[i], kNone);
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = __builtin_fma(d[i], 1.4426950408889634, kRound);
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = __builtin_fma(t[i] - kRound, -0.6931471805599453, d[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __builtin_fma(2.473298746639189e-05, d[i], C[0]);
#pragma unroll
    for (int k = 1; k < 8; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = __builtin_fma(y[i], d[i], C[k]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u32x2_t u = __builtin_bit_cast(u32x2_t, y[i]);
        u[1] += __builtin_bit_cast(u32x2_t, t[i])[0] << 20;
        e[i] = __builtin_bit_cast(double, u);
    }
}
__device__ __forceinline__ double exp_over(float x, float m, double inv_t) {
    double e;
    exp_over<1>(&x, m, inv_t, &e);
    return e;
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

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

constexpr int kPer = kVerifyBlock / 64;  // values of a lane in a block: 4 j + u is the block's 256 j + 4 lane + u
constexpr int kBad = 0x7fffffff;

// A block of a row (what is past its end comes as 0): loads without a branch of a lane's
// own, so that a wave works on one block while the next one's are under way.
__device__ __forceinline__ void load_block(float (&v)[kPer], uint64_t row, int block, int n) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uniform_u64(row)), (short)0, n * 4, kBufferWord3);
    const int at = (block * kVerifyBlock + 4 * lane_id()) * 4;
    if ((block + 1) * kVerifyBlock <= n) {
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            const f32x4_t w = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, at + 1024 * j, 0, 0));
#pragma unroll
            for (int u = 0; u < 4; ++u) v[4 * j + u] = w[u];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            v[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, at + 1024 * (i / 4) + 4 * (i % 4), 0, 0));
    }
}
// Logits past the row's end: -infinity.
__device__ __forceinline__ void end_block(float (&v)[kPer], int block, int n) {
    if ((block + 1) * kVerifyBlock <= n) return;
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = block * kVerifyBlock + 256 * (i / 4) + 4 * lane_id() + i % 4 < n ? v[i] : -INFINITY;
}

// The place in a block where the sums of the weights, `before` what went before them, pass
// thr; at rounding's edge the last above `least`, -1 where none is.  weights(j, e): the
// lane's four of part j.
template <typename F>
__device__ __forceinline__ int find_in_block(const F& weights, double before, double thr, double least) {
    constexpr int N = kPer / 4;
    double t[N], incl[N], e[4];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        weights(j, e);
        t[j] = (e[0] + e[1]) + (e[2] + e[3]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) incl[j] = scan_f64(t[j]);
    int in = -1, lane = 0;
    double from = 0.0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint64_t some = __ballot(t[j] > kOfFour * least), hit = __ballot(before + incl[j] > thr && t[j] > kOfFour * least);
        if (some) in = j, lane = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some), from = before + incl[j] - t[j];
        if (hit) break;
        before += lane_f64(incl[j], 63);
    }
    if (in < 0) return -1;
    weights(in, e);
    int u = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (u >= 0 && from > thr) continue;  // found
        from += e[k];
        if (e[k] > least) u = k;
    }
    return 256 * in + 4 * lane + __builtin_amdgcn_readlane(u, lane);
}
// Part j of the lane's values.
__device__ __forceinline__ void part_of(const float (&v)[kPer], int j, float (&x)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        x[u] = v[u];
#pragma unroll
        for (int k = 1; k < kPer / 4; ++k) x[u] = j == k ? v[4 * k + u] : x[u];
    }
}

// A row's blocks in LDS, for one wave.
struct Room {
    double w[kVerifyBlocks];  // their sums
    float m[kVerifyBlocks];
};

// Which of a row's blocks holds the border: their sums in order, and `share` of the whole.
// The border and what goes before the block are left in thr and before; -1 where no sum
// holds a weight above `least`.
__device__ __forceinline__ int find_block(const double* w, int blocks, double share, double least, double& thr, double& before) {
    double all = 0.0;
    for (int i = lane_id(); i - lane_id() < blocks; i += 64) all += i < blocks ? w[i] : 0.0;
    thr = share * wave_sum_f64(all);
    int at = -1;
    double done = 0.0;
    before = 0.0;
    for (int i0 = 0; i0 < blocks; i0 += 64) {
        const double x = i0 + lane_id() < blocks ? w[i0 + lane_id()] : 0.0, incl = done + scan_f64(x);
        const uint64_t some = __ballot(x > kOfBlock * least), hit = __ballot(incl > thr && x > kOfBlock * least);
        done = lane_f64(incl, 63);
        if (!some) continue;
        const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
        at = i0 + l, before = lane_f64(incl - x, l);
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

// The records of a part of row t (those of slot `slot`), by the whole workgroup of WAVES: the block's
// sum (NaN: a logit is NaN or infinite), its largest logit, and the first id of that.
template <int WAVES>
__device__ __forceinline__ void scan_part(const VerifyArgs& a, const Seq& s, int t, int slot, int part) {
    const int wave = wave_id(), end = min(a.blocks, (part + 1) * a.per_part);
    const uint64_t row = logits_row(a, t);
    float x[kPer], next[kPer];
    int blk = part * a.per_part + wave;
    if (blk < end) load_block(next, row, blk, a.vocab);
    for (; blk < end; blk += WAVES) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = next[i];
        if (blk + WAVES < end) load_block(next, row, blk + WAVES, a.vocab);
        end_block(x, blk, a.vocab);
        float mx = x[0];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) mx = fmaxf(mx, x[i]), bad |= !(x[i] < INFINITY);
        mx = wave_top(mx);
        double sum = 0.0;
        int id = kBad;
        if (s.temp > 0.0f) {
            double some[4] = {};
#pragma unroll
            for (int i = 0; i < kPer; i += 4) {
                double e[4];
                exp_over<4>(x + i, mx, s.inv_t, e);
#pragma unroll
                for (int u = 0; u < 4; ++u) some[u] += e[u];
            }
            sum = wave_sum_f64((some[0] + some[1]) + (some[2] + some[3]));
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

// A row's records joined by a wave, the blocks' sums relative to the row's largest logit left
// in `room`.
struct Row {
    float m;    // the largest logit
    double s;   // the sum relative to it, NaN for a row from which nothing can be drawn
    int first;  // the first id of the largest logit
};
__device__ __forceinline__ Row join_row(const VerifyArgs& a, const Seq& s, int slot, Room& room) {
    Row r{-INFINITY, 0.0, kBad};
    float mx = -INFINITY;
    int id = kBad;
    constexpr int N = 4;  // loads at a time
    for (int b0 = lane_id(); b0 - lane_id() < a.blocks; b0 += 64 * N) {
        uint64_t w[N], mi[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t at = record(a, slot, min(b0 + 64 * i, a.blocks - 1));
            w[i] = get64(at), mi[i] = get64(at + 8);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int blk = b0 + 64 * i;
            if (blk >= a.blocks) continue;
            const float m = __uint_as_float((uint32_t)mi[i]);
            room.w[blk] = __builtin_bit_cast(double, w[i]), room.m[blk] = m;
            if (m > mx) mx = m, id = (int)(mi[i] >> 32);  // blocks rise: the first of equal ones stays
        }
    }
    r.m = wave_top(mx);
    r.first = wave_least(mx == r.m ? id : kBad);
    double sum = 0.0;
    for (int blk = lane_id(); blk < a.blocks; blk += 64) {
        double w = room.w[blk];
        if (s.temp > 0.0f) w *= exp_over(room.m[blk], r.m, s.inv_t);
        room.w[blk] = w;
        sum += w;
    }
    r.s = r.m == -INFINITY ? __builtin_nan("") : wave_sum_f64(sum);
    return r;
}

// The first token of row t that can be drawn.  (A border of 0 lies below all sums, also those of
// tokens that can't be; the numbers above 0 are 2^-149 at least, beside which a row's 2^19 such
// weights are nothing, so that only 0 has to look at each.)
__device__ __forceinline__ int draw_first(const VerifyArgs& a, const Seq& s, int t, const Row& r, const Room& room) {
    for (int b0 = 0; b0 < a.blocks; b0 += 64) {
        const int i = b0 + lane_id();
        const uint64_t some = __ballot(i < a.blocks && exp_over(room.m[min(i, a.blocks - 1)], r.m, s.inv_t) > kNothing);
        if (!some) continue;
        const int blk = b0 + __builtin_ctzll(some);
        float x[kPer];
        load_block(x, logits_row(a, t), blk, a.vocab);
        end_block(x, blk, a.vocab);
        int id = kBad;
#pragma unroll 1
        for (int j = kPer / 4 - 1; j >= 0; --j) {
            float y[4];
            double e[4];
            part_of(x, j, y);
            exp_over<4>(y, r.m, s.inv_t, e);
#pragma unroll
            for (int u = 3; u >= 0; --u) id = e[u] > kNothing ? blk * kVerifyBlock + 256 * j + 4 * lane_id() + u : id;
        }
        return wave_least(id);
    }
    return -1;
}

// The token of row t that number u draws, -1: none can be.
__device__ __forceinline__ int draw(const VerifyArgs& a, const Seq& s, int t, const Row& r, const Room& room, float u) {
    if (r.s != r.s) return -1;
    if (s.temp == 0.0f) return r.first;
    double thr, before;
    float x[kPer];
    if (!(u > 0.0f)) return draw_first(a, s, t, r, room);
    const int blk = find_block(room.w, a.blocks, (double)u, kNothing, thr, before);
    if (blk < 0) return -1;
    load_block(x, logits_row(a, t), blk, a.vocab);
    end_block(x, blk, a.vocab);
    auto weights = [&](int j, double (&e)[4]) {
        float y[4];
        part_of(x, j, y);
        exp_over<4>(y, r.m, s.inv_t, e);
    };
    const int at = find_in_block(weights, before, thr, kNothing);
    return at < 0 ? -1 : blk * kVerifyBlock + at;
}

// What is left of a row: max(p - taken q, 0), four at a time.  What can't be drawn comes as 0,
// since kNothing is taken off, which is less than the last bit of any but the smallest.
struct Left {
    float m;
    double inv_s, inv_t, taken;
    __device__ __forceinline__ void operator()(const float (&x)[4], const float (&q)[4], double (&e)[4]) const {
        exp_over<4>(x, m, inv_t, e);
#pragma unroll
        for (int u = 0; u < 4; ++u) e[u] = fmax(__builtin_fma(-taken, (double)q[u], __builtin_fma(e[u], inv_s, -kNothing * inv_s)), 0.0);
    }
};
__device__ __forceinline__ void load_both(const VerifyArgs& a, int t, int blk, float (&x)[kPer], float (&q)[kPer]) {
    load_block(x, logits_row(a, t), blk, a.vocab);
    load_block(q, probs_row(a, t), blk, a.vocab);
    end_block(x, blk, a.vocab);
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
            const double e = exp_over(x, st.m, s.inv_t);
            fits = e > kNothing && (double)u * (double)q < e / st.s;
        } else {
            fits = token == st.z;
        }
    }
};

// A sequence's walk, by one wave, from node st.cur on until its end (true) or until what is
// left of a row has to be summed (false; then, with the blocks' sums in `room`, the walk goes on).
__device__ __forceinline__ bool walk(const VerifyArgs& a, const Seq& s, int b, VerifyState& st, Room& room) {
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
                const double e = exp_over(gptr<float>(logits_row(a, t))[d], m, s.inv_t), p = __builtin_fma(-st.taken, q, e / S);
                if (e > kNothing && p > 0.0 && u * q * st.left < p) {
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
                const Row r = join_row(a, s, t, room);
                next = draw(a, s, t, r, room, u);
            } else {
                double thr, before;
                float x[kPer], q[kPer];
                const int blk = max(0, find_block(room.w, a.blocks, (double)u, 0.0, thr, before));
                load_both(a, t, blk, x, q);
                const Left left{m, 1.0 / S, s.inv_t, st.taken};
                auto weights = [&](int j, double (&e)[4]) {
                    float y[4], z[4];
                    part_of(x, j, y), part_of(q, j, z);
                    left(y, z, e);
                };
                next = blk * kVerifyBlock + max(0, find_in_block(weights, before, thr, 0.0));
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
//
// 26 rows of 151,936 logits 14.5 us: the launch, two blocks a wave, the join, the draw and the
// walk, one behind the other.  116 rows 31 us, 600 rows 119: 3.1 TB/s; loads alone took 93, and the
// exponentials' 18 instructions a logit are 51 more, half of which the four waves of a SIMD hide.
extern "C" __global__ void __launch_bounds__(256, 4) lp_verify_rows(const VerifyArgs a) {
    __shared__ Room room;
    const int t = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - t * a.parts, wave = wave_id();
    const int b = sequence_of_row(a, t);
    if (blockIdx.x == 0 && wave == 3)  // sequences without a token, or where no row has a sequence all
        for (int i = lane_id(); i < a.batch; i += 64) {
            if (b < a.batch && seq_of(a, i).n > 0) continue;
            for (int j = 0; j <= a.max_depth; ++j) gptr_w<int>(a.path)[(uint64_t)(uint32_t)i * (uint32_t)(a.max_depth + 1) + (uint32_t)j] = -1;
            gptr_w<int>(a.kept)[i] = 0, gptr_w<int>(a.next)[i] = -1;
            if (a.probs) gptr_w<VerifyState>(a.state)[i].pending = 0;
        }
    if (b >= a.batch) return;  // whole workgroups, here and below
    const Seq s = seq_of(a, b);
    if (t < s.t0 || t - s.t0 >= s.n) return;
    scan_part<4>(a, s, t, t, part);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (wave) return;
    if (a.parts > 1 && !last_of(a, t, a.parts)) return;
    const Row r = join_row(a, s, t, room);
    const bool sampled = a.probs && s.temp > 0.0f;
    put_stat(a, t, r, sampled ? -1 : draw(a, s, t, r, room, gptr<float>(a.uniforms)[t]));
    if (!last_of(a, a.row_counters + b, s.n)) return;
    VerifyState st{0, 0, 1, 0, 0.0, 1.0};
    put_node(a, b, 0, 0);
    walk(a, s, b, st, room);
    if (a.probs && lane_id() == 0) gptr_w<VerifyState>(a.state)[b] = st;
}

// What is left of a row, for the sequences whose walk stands there: workgroup (sequence,
// part) sums a wave's blocks, the last one goes on with the walk, and where that needs
// another row's or more taken from this one, sums that alone.  32 chains of 6 nodes, 151,936
// logits: 12 us for 39 MB, mostly one chain: a wave's blocks, the arrival, the walk and its draw.
// Trees turn down several: one of 26 nodes, 4 turned down, 97 us, about 30 each behind the first.
extern "C" __global__ void __launch_bounds__(64 * kVerifyWaves) lp_verify_left(const VerifyArgs a) {
    __shared__ Room room;
    __shared__ VerifyState now;
    __shared__ int flag;
    const int b = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - b * a.parts;
    const int wave = wave_id(), lane = lane_id();
    VerifyState st = gptr<VerifyState>(a.state)[b];
    if (!st.pending) return;  // whole workgroups, here and below
    const Seq s = seq_of(a, b);
    const uint64_t mine = a.left + (uint64_t)(uint32_t)b * (uint32_t)a.blocks * 8;
    auto sum_block = [&](int blk) {
        float x[kPer], q[kPer];
        load_both(a, s.t0 + st.cur, blk, x, q);
        const Stat r = get_stat(a, s.t0 + st.cur);
        const Left left{r.m, 1.0 / r.s, s.inv_t, st.taken};
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            float y[4], z[4];
            double e[4];
            part_of(x, j, y), part_of(q, j, z);
            left(y, z, e);
            sum += (e[0] + e[1]) + (e[2] + e[3]);
        }
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
    for (int i = threadIdx.x; i < a.blocks; i += 64 * kVerifyWaves) room.w[i] = getf64(mine + 8 * i);
    for (;;) {
        __syncthreads();
        if (wave == 0) {
            double z = 0.0;
            for (int i = lane; i < a.blocks; i += 64) z += room.w[i];
            st.left = wave_sum_f64(z), st.pending = 0;
            const bool done = walk(a, s, b, st, room);
            if (lane == 0) now = st, flag = done;
        }
        __syncthreads();
        if (flag) return;
        st = now;
        for (int blk = wave; blk < a.blocks; blk += kVerifyWaves) {
            const double sum = sum_block(blk);
            if (lane == 0) room.w[blk] = sum;
        }
    }
}

// The rows of the path alone, chosen drafts: `parts` workgroups a sequence share the row
// that the walk stands at.  Each takes a group of its blocks (the count of those that are
// taken, beside the node's number); who ends a row's last group joins it, goes a node down
// and says so, and all take groups of that one.  Nobody needs another one to go on: who finds
// no group left looks for the next node for a while and leaves, and who ended the last
// group is there to take all of the next row's if need be.  The last one to leave clears the words.
//
// 32 trees of up to 60 nodes, at most 6 of them kept, 151,936 logits: 67 us; a node is about
// 11, of which 3 to 5 are the row's blocks, 4 the join and the draw, 2 word that it is done
// (a launch for each node 75 us, half of a node's the launch; the words 64 bytes apart and
// workgroups of four waves 103 us: many look at one memory channel).
constexpr int kTaken = 0, kEnded = 1, kGone = 2, kLen = 3;  // words of a sequence
constexpr int kOver = 0x7fff;                               // no node
constexpr int kLooks = 64;                                  // about a microsecond each

extern "C" __global__ void __launch_bounds__(64 * kPathWaves, 4) lp_verify_path(const VerifyArgs a) {
    __shared__ Room room;
    __shared__ int share, fell[kPathWaves];
    const int b = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - b * a.parts, wave = wave_id();
    const Seq s = seq_of(a, b);
    if (s.n <= 0) {
        if (part == 0 && wave == 0) put_end(a, b, 0, -1);
        return;  // whole workgroups
    }
    int* const word = reinterpret_cast<int*>(a.sync) + (uint64_t)(uint32_t)(b * a.row_counters) * kPagedStride;
    int up = -1, token = -1;  // of the first 64 nodes, one a lane
    if (lane_id() < s.n) up = gptr<int>(a.parents)[s.t0 + lane_id()], token = gptr<int>(a.drafts)[s.t0 + lane_id()];
    // where the starts do not rise no row has a sequence, as in lp_verify_rows: seen by the
    // other waves while the first one waits for its group (by that one, or by who ends the
    // root's row, 0.9 to 1.5 us more)
    if (wave) {
        bool falls = false;
        for (int i = 64 * (wave - 1) + lane_id(); i < a.batch; i += 64 * (kPathWaves - 1)) falls |= gptr<int>(a.q_starts)[i + 1] < gptr<int>(a.q_starts)[i];
        const bool some = __ballot(falls) != 0;
        if (lane_id() == 0) fell[wave] = some;
    }
    for (;;) {
        if (threadIdx.x == 0) {
            int c = atomicAdd(word + kTaken, 1);
            for (int look = 0; (c & 0xffff) >= a.parts && c >> 16 != kOver;) {
                const int now = agent_load(word + kTaken);
                if (now >> 16 != c >> 16)
                    c = now >> 16 == kOver ? now : atomicAdd(word + kTaken, 1);
                else if (++look == kLooks)
                    c = kOver << 16;
                else
                    __builtin_amdgcn_s_sleep(2);
            }
            share = c;
        }
        __syncthreads();
        const int c = __builtin_amdgcn_readfirstlane(share), cur = c >> 16, t = s.t0 + cur;
        if (cur == kOver) break;
        const float u = gptr<float>(a.uniforms)[t];
        scan_part<kPathWaves>(a, s, t, b, c & 0xffff);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (wave) continue;
        int ended = 0;
        if (lane_id() == 0) ended = atomicAdd(word + kEnded, 1);
        if (__builtin_amdgcn_readfirstlane(ended) != a.parts - 1) continue;
        const int len = agent_load(word + kLen);
        const Row r = join_row(a, s, b, room);
        const int z = draw(a, s, t, r, room, u);
        const bool none = __ballot(lane_id() > 0 && lane_id() < kPathWaves && fell[lane_id() % kPathWaves]) != 0;
        int to = -1;
        if (z >= 0 && len < a.max_depth && !none)
            for (int i0 = cur & ~63; i0 < s.n && to < 0; i0 += 64) {
                const int i = i0 + lane_id();
                int p = up, d = token;
                if (i0) {
                    p = d = -1;
                    if (i < s.n) p = gptr<int>(a.parents)[s.t0 + i], d = gptr<int>(a.drafts)[s.t0 + i];
                }
                const uint64_t fit = __ballot(i > cur && p == cur && d == z);
                if (fit) to = i0 + __builtin_ctzll(fit);
            }
        if (lane_id() == 0) {
            agent_store(word + kEnded, 0);
            agent_store(word + kLen, len + 1);
            __builtin_amdgcn_s_waitcnt(0);
            atomicExch(word + kTaken, (to < 0 ? kOver : to) << 16);
        }
        if (!none) put_node(a, b, len, cur);
        if (to < 0) put_end(a, b, none ? 0 : len + 1, none ? -1 : z);
    }
    if (threadIdx.x == 0 && atomicAdd(word + kGone, 1) == a.parts - 1)
        for (int i = 0; i < 4; ++i) agent_store(word + i, 0);
}
