// gfx950 kernels of a batch's KV cache in pages: the new tokens' queries and
// keys normed per head and rotated with keys and values written into their
// pages (lp_kv_append_*), and attention of one or many new tokens a sequence
// over its pages (lp_attn_few_*, lp_attn_many_* and lp_attn_join_*).
//
// A page holds page_rows rows of one KV head, as fp16 [page_rows, head_dim] or
// as a q4 region (f16 scales [page_rows, head_dim / 32], then nibbles
// [page_rows, head_dim / 2], value q stored as q + 8).  Page p of KV head g is
// at base + (p kv_heads + g) page_bytes; row r of sequence b is row
// r % page_rows of page table[b][r / page_rows].
#include "lp_device.h"

using namespace lp;
using namespace lpk;

namespace {

// ---- pages --------------------------------------------------------------------

template <int D, bool Q4>
__device__ __forceinline__ uint64_t page_at(const PagedCache& c, uint64_t base, int page, int head) {
    return base + ((uint64_t)page * (uint32_t)c.kv_heads + (uint32_t)head) * (uint32_t)page_bytes(D, 1 << c.page_log2, Q4);
}

// The page of a sequence's row, or -1: past the table's width, or an entry
// that names no page of the pool.
__device__ __forceinline__ int page_of(const PagedCache& c, int b, int row) {
    const int col = row >> c.page_log2;
    if (row < 0 || col >= c.max_pages) return -1;
    const int p = gptr<int>(c.table)[(uint64_t)b * (uint32_t)c.max_pages + (uint32_t)col];
    return (uint32_t)p < (uint32_t)c.pages ? p : -1;
}

// ---- 64-bit values across lanes -------------------------------------------------

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)lo | (uint64_t)(uint32_t)hi << 32);
}

// over each row of 16 lanes: neighbours, pairs, the halves of eight, the halves
template <typename Op>
__device__ __forceinline__ double row16_f64(double v, Op op) {
    v = op(v, dpp_f64<0xb1>(v));
    v = op(v, dpp_f64<0x4e>(v));
    v = op(v, dpp_f64<0x141>(v));
    return op(v, dpp_f64<0x140>(v));
}

// d > 0 to 7 significant bits, ties to even.
__device__ __forceinline__ double round7(double d) {
    uint64_t b = __builtin_bit_cast(uint64_t, d);
    b += (1ull << 45) - 1 + (b >> 46 & 1);
    return __builtin_bit_cast(double, b >> 46 << 46);
}

// 1 / sqrt(a), a > 0: the fp32 one and two Newton steps, 2^-24 -> 2^-47 -> 64 bits.
// (a far from 1 is brought into fp32's range by the powers of two of its exponent.)
__device__ __forceinline__ double rsqrt_f64(double a) {
    const int e = __builtin_amdgcn_frexp_exp(a) & ~1;
    const double m = __builtin_amdgcn_ldexp(a, -e);  // 0.5 .. 2
    double y = (double)__builtin_amdgcn_rsqf((float)m);
    y = __builtin_fma(0.5 * y, __builtin_fma(-m * y, y, 1.0), y);
    y = __builtin_fma(0.5 * y, __builtin_fma(-m * y, y, 1.0), y);
    return __builtin_amdgcn_ldexp(y, -e / 2);
}

// x / d with inv = 1 / d to a unit or so: the quotient corrected by its
// remainder, so that one that is a number of 53 bits comes out as it.
__device__ __forceinline__ double div_by(double x, double d, double inv) {
    const double q = x * inv;
    return __builtin_fma(__builtin_fma(-q, d, x), inv, q);
}

// 1 / s, s of 7 significant bits within the normal fp32 numbers.
__device__ __forceinline__ double rcp_f64(double s) {
    double y = (double)__builtin_amdgcn_rcpf((float)s);
    y = __builtin_fma(__builtin_fma(-s, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-s, y, 1.0), y, y);
}

// sin and cos of r, |r| <= pi: Taylor's series about the nearest multiple of
// pi / 2, whose first term left out is below 2^-53 there.
__device__ __forceinline__ void sincos_f64(double r, double& sn, double& cs) {
    const double k = rint(r * 0.63661977236758138);
    const double x = __builtin_fma(-k, 6.1232339957367660e-17, __builtin_fma(-k, 1.5707963267948966, r));
    const double z = x * x;
    auto by_z = [&](double y, double c0) { return __builtin_fma(y, z, c0); };
    double s = by_z(-7.6471637318198164e-13, 1.6059043836821613e-10);  // 1 / 15!, 1 / 13!, ...
    s = by_z(s, -2.5052108385441720e-8);
    s = by_z(s, 2.7557319223985893e-6);
    s = by_z(s, -1.9841269841269841e-4);
    s = by_z(s, 8.3333333333333333e-3);
    s = by_z(s, -0.16666666666666667);
    s = by_z(s, 1.0);
    double c = by_z(4.7794773323873853e-14, -1.1470745597729725e-11);  // 1 / 16!, 1 / 14!, ...
    c = by_z(c, 2.0876756987868099e-9);
    c = by_z(c, -2.7557319223985888e-7);
    c = by_z(c, 2.4801587301587302e-5);
    c = by_z(c, -1.3888888888888889e-3);
    c = by_z(c, 4.1666666666666667e-2);
    c = by_z(c, -0.5);
    c = by_z(c, 1.0);
    s *= x;
    const int q = (int)k & 3;
    const double a = q & 1 ? c : s, b = q & 1 ? s : c;
    sn = q & 2 ? -a : a;
    cs = (q + 1) & 2 ? -b : b;
}

// The token's sequence: the sequences that end at or before it (batch for a token
// behind the last one; a token before the first one's start is none of sequence 0's).
__device__ __forceinline__ int sequence_of(uint64_t q_starts, int batch, int token) {
    int b = 0;
    for (int i = 0; i < batch; i += 64) {
        const int at = i + lane_id();
        const bool past = at < batch && gptr<int>(q_starts)[at + 1] <= token;
        b += __popcll(__ballot(past));
    }
    return __builtin_amdgcn_readfirstlane(b);
}

// ---------------------------------------------------------------------------
// Append.  A token's rows are its query heads, its key heads and its value
// heads, D floats each; D / 4 lanes take a row, lane j the columns 2j, 2j + 1
// and the pair partners D/2 + 2j, D/2 + 2j + 1, so a rotation stays in the
// lane and a q4 group of 32 columns is one row of 16 lanes.  `parts` waves
// share a token's rows; the angles are made once per wave.
//
// Everything up to the last rounding is in 64 bits: the angle pos inv_freq of a
// far position needs it, and a 4-bit code then is that of the exact value
// whatever the order of the sums.  Vector fp64 runs at fp32's rate here, but
// its divisions, square roots and sines are long: they are short series and
// Newton steps from fp32 (2,404 tokens of 32 + 2 x 4 heads into 4-bit pages, 100
// MB in all: 41 us with the library's, 27.4 with these, 3.6 TB/s).
// ---------------------------------------------------------------------------
// (by value: a choice between members of a block makes the compiler keep it in memory)
__device__ __forceinline__ uint64_t pick(bool c, uint64_t a, uint64_t b) { return c ? a : b; }

template <int D, bool Q4>
__device__ __forceinline__ void append_body(const KvAppendPagedArgs& a) {
    constexpr int LPR = D / 4, RPW = 64 / LPR, G = D / 32;
    const int lane = lane_id(), j = lane % LPR, sub = lane / LPR;
    const int w = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    const int token = w / a.parts;
    if (token >= a.tokens) return;  // whole waves
    const int b = sequence_of(a.q_starts, a.batch, token);
    // before the first sequence or behind the last: left as it was
    if (b >= a.batch || token < gptr<int>(a.q_starts)[b]) return;
    const int pos = gptr<int>(a.seq_lens)[b] - (gptr<int>(a.q_starts)[b + 1] - token);
    const int page = page_of(a.c, b, pos), prow = pos & ((1 << a.c.page_log2) - 1);
    // pos inv_freq in radians, less whole turns (2 pi in two parts)
    double cs[2], sn[2];
    const float2 fr = gptr<float2>(a.inv_freq)[j];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const double ang = (double)pos * (double)(u ? fr.y : fr.x);
        const double k = rint(ang * 0.15915494309189535);
        const double r = __builtin_fma(-k, 2.4492935982947064e-16, __builtin_fma(-k, 6.283185307179586, ang));
        sincos_f64(r, sn[u], cs[u]);
        cs[u] *= (double)a.mscale;
        sn[u] *= (double)a.mscale;
    }
    const int H = a.heads, KV = a.c.kv_heads, rows = H + 2 * KV;
    const int r1 = min(rows, (w % a.parts + 1) * a.rows_per_part);
    const uint64_t qt = a.q + (uint64_t)token * (uint32_t)a.q_stride * 4, kt = a.k + (uint64_t)token * (uint32_t)a.k_stride * 4;
    const uint64_t vt = a.v + (uint64_t)token * (uint32_t)a.v_stride * 4;
    const uint64_t qw = a.q_norm, kw = a.k_norm, kout = a.k_out, vout = a.v_out;
    const uint64_t kpage = page_at<D, Q4>(a.c, a.c.k_pages, max(page, 0), 0), vpage = page_at<D, Q4>(a.c, a.c.v_pages, max(page, 0), 0);
    // a row's floats and its norm's weights; the next rows' are on their way
    // while these are worked on
    float2 f0, f1, w0, w1;
    auto load = [&](int row) {
        f0 = f1 = make_float2(0.0f, 0.0f), w0 = w1 = make_float2(1.0f, 1.0f);
        if (row >= r1) return;
        const bool isq = row < H, isk = !isq && row < H + KV;
        const int head = isq ? row : isk ? row - H : row - H - KV;
        const uint64_t src = pick(isq, qt, pick(isk, kt, vt)) + (uint32_t)(head * D * 4);
        f0 = gptr<float2>(src)[j];
        f1 = gptr<float2>(src)[LPR + j];
        const uint64_t nw = pick(isq, qw, pick(isk, kw, 0));
        if (nw) {
            w0 = gptr<float2>(nw)[j];
            w1 = gptr<float2>(nw)[LPR + j];
        }
    };
    const int rfirst = w % a.parts * a.rows_per_part;
    load(rfirst + sub);
    for (int r = rfirst; r < r1; r += RPW) {
        const int row = r + sub;
        const bool on = row < r1, isq = row < H, isk = !isq && row < H + KV;
        const int head = isq ? row : isk ? row - H : row - H - KV;
        double x[4] = {f0.x, f0.y, f1.x, f1.y};
        const double wt[4] = {w0.x, w0.y, w1.x, w1.y};
        load(row + RPW);
        double ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
        ss = row16_f64(ss, [](double p, double q) { return p + q; });
        if constexpr (LPR == 32) ss += __shfl_xor(ss, 16, 64);
        if (isq || isk) {
            if (pick(isq, qw, kw)) {
                const double inv = rsqrt_f64(ss / (double)D + (double)a.eps);
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] *= inv * wt[u];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const double p = x[u], q = x[u + 2];
                x[u] = p * cs[u] - q * sn[u];
                x[u + 2] = p * sn[u] + q * cs[u];
            }
        }
        if (on && isq) {
            const uint64_t dst = a.q_out + ((uint64_t)token * (uint32_t)a.q_out_stride + (uint32_t)(head * D)) * 4;
            gptr_w<float2>(dst)[j] = make_float2((float)x[0], (float)x[1]);
            gptr_w<float2>(dst)[LPR + j] = make_float2((float)x[2], (float)x[3]);
        }
        if (!__ballot(on && !isq)) continue;  // queries only
        float2 held[2];
        const uint64_t pg = pick(isk, kpage, vpage) + (uint32_t)(isq ? 0 : head) * (uint32_t)page_bytes(D, 1 << a.c.page_log2, Q4);
        const bool store = on && !isq && page >= 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const double x0 = x[2 * u], x1 = x[2 * u + 1];
            if constexpr (Q4) {
                // the group's scale; a NaN counts as zero, so that a 4-bit row holds numbers only
                const double m = row16_f64(fmax(fmax(fabs(x0), fabs(x1)), 0.0), [](double p, double q) { return fmax(p, q); });
                const double s = fmax(round7(div_by(fmin(m, 7.0 * kQ4MaxScale), 7.0, 1.0 / 7.0)), kQ4MinScale), is = rcp_f64(s);
                auto code = [&](double y) {  // (8 scales are cut as 7 are: no infinities from here)
                    return y == y ? (int)fmin(fmax(rint(div_by(fmin(fmax(y, -8.0 * s), 8.0 * s), s, is)), -7.0), 7.0) : 0;
                };
                const int c0 = code(x0), c1 = code(x1);
                held[u] = make_float2((float)(c0 * s), (float)(c1 * s));
                // eight columns' nibbles meet in a word
                uint32_t n = (uint32_t)((c0 + 8) | (c1 + 8) << 4) << (8 * (lane & 3));
                n |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, 0xb1, 0xf, 0xf, false);
                n |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)n, 0x4e, 0xf, 0xf, false);
                if (store) {
                    const int g = u * (G / 2) + j / 16;
                    if ((j & 15) == 0)
                        gptr_w<uint16_t>(pg)[prow * G + g] = __builtin_bit_cast(uint16_t, (_Float16)(float)s);
                    if ((j & 3) == 0)
                        gptr_w<uint32_t>(pg + (uint32_t)(2 * G << a.c.page_log2))[prow * (D / 8) + u * (D / 16) + j / 4] = n;
                }
            } else {
                const _Float16 h0 = (_Float16)x0, h1 = (_Float16)x1;
                held[u] = make_float2((float)h0, (float)h1);
                if (store)
                    gptr_w<uint32_t>(pg)[prow * (D / 2) + u * LPR + j] =
                        (uint32_t)__builtin_bit_cast(uint16_t, h0) | (uint32_t)__builtin_bit_cast(uint16_t, h1) << 16;
            }
        }
        const uint64_t ko = pick(isk, kout, vout);
        if (on && !isq && ko) {
            const uint64_t dst = ko + ((uint64_t)token * (uint32_t)KV + (uint32_t)head) * (D * 4);
            gptr_w<float2>(dst)[j] = held[0];
            gptr_w<float2>(dst)[LPR + j] = held[1];
        }
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_kv_append_f16_d64(const KvAppendPagedArgs a) { append_body<64, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_f16_d128(const KvAppendPagedArgs a) { append_body<128, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_q4_d64(const KvAppendPagedArgs a) { append_body<64, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_q4_d128(const KvAppendPagedArgs a) { append_body<128, true>(a); }

namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef int v2i32_t __attribute__((ext_vector_type(2)));

#define LP_LDS __attribute__((address_space(3)))
// LDS bytes are written as one type and read as another
typedef uint16_t u16_any __attribute__((may_alias));
typedef uint32_t u32_any __attribute__((may_alias));
typedef uint64_t u64_any __attribute__((may_alias));
typedef u32x4_t u32x4_any __attribute__((may_alias));
typedef f32x4_t f32x4_any __attribute__((may_alias));
typedef float f32_any __attribute__((may_alias));
typedef float2 float2_any __attribute__((may_alias));

__device__ __forceinline__ f32x4_t mfma16(const u32x4_t& a, const u32x4_t& b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Two values as fp16, cut towards zero, and what that leaves out of each, rounded
// to fp16 (one mixed multiply-add each): 2^-22 of a value is left out, or 2^-25
// where that is more.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    const half2_t x = __builtin_bit_cast(half2_t, h);
    float minus;  // behind the asm lest -1 x + a become a subtraction of its own
    asm("" : "=s"(minus) : "0"(-1.0f));
    half2_t y;
    y[0] = (_Float16)__builtin_fmaf((float)x[0], minus, a), y[1] = (_Float16)__builtin_fmaf((float)x[1], minus, b);
    lo = __builtin_bit_cast(uint32_t, y);
}

// Eight nibbles times their scales: pairs (n0, n4), (n1, n5), (n2, n6), (n3, n7)
// of q + 8, each pair by s (scales of its two) with c = -72 s.
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, half2_t s, half2_t c) {
    const half2_t v = __builtin_bit_cast(half2_t, and_or(w, 0x00f000f0u, 0x54005400u));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(v, s, c));
}
__device__ __forceinline__ u32x4_t nibbles8(uint32_t w, const half2_t (&s)[4], const half2_t (&c)[4]) {
    u32x4_t r;
    r[0] = nibble_pair(w << 4, s[0], c[0]);
    r[1] = nibble_pair(w, s[1], c[1]);
    r[2] = nibble_pair(w >> 4, s[2], c[2]);
    r[3] = nibble_pair(w >> 8, s[3], c[3]);
    return r;
}

// Probabilities are held relative to a base kLift powers of two below the maximum that
// was current when it was set, which a score may pass by kSlack more before the base
// is raised: the largest is near 2^kLift and none is above 2^15, an image's reach.  What
// the images leave out of a small one is then 2^-34 of the largest at most (with the
// maximum for a base 2^-25, of one 17 nats below it a third).
// A wider lift raises the base more often (38 tokens of 12 sequences: 40.3 us, with
// kLift 11 and kSlack 4 41.2).
constexpr float kLift = 9.0f, kSlack = 6.0f;

__device__ __forceinline__ bool odd_halves(uint32_t w) {  // a NaN or infinity among the two
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}

// The new tokens of sequence b and its rows, as the kernels take them.
struct SeqView {
    int t0, n, len;  // first token, tokens (at most max_q), rows
    int p0;          // the first token's position
};
__device__ __forceinline__ SeqView seq_view(const AttnPagedArgs& a, int b) {
    SeqView s;
    s.t0 = gptr<int>(a.q_starts)[b];
    const int n = gptr<int>(a.q_starts)[b + 1] - s.t0;
    s.len = min(gptr<int>(a.seq_lens)[b], a.max_seq);
    s.p0 = s.len - n;
    s.n = min(n, a.max_q);
    if (s.t0 < 0 || s.t0 > a.tokens - s.n) s.n = 0;  // starts that name no tokens
    return s;
}

// The rows that a query row of the sequence sees.
__device__ __forceinline__ int seen_rows(const AttnPagedArgs& a, const SeqView& s, int row) {
    return max(0, min(s.p0 + row / a.group + 1, s.len));
}

// A sequence's rows of one KV head per split, and the record of (sequence and
// KV head bg, split, query row): D sums, then {maximum, sum} behind all of them.
__device__ __forceinline__ uint64_t rec_index(const AttnPagedArgs& a, int bg, int split, int row) {
    return ((uint64_t)(uint32_t)bg * (uint32_t)a.splits + (uint32_t)split) * (uint32_t)a.rows + (uint32_t)row;
}
template <int D>
__device__ __forceinline__ uint64_t rec_sums(const AttnPagedArgs& a) {
    return a.part + (uint64_t)(uint32_t)(a.batch * a.c.kv_heads) * (uint32_t)a.splits * (uint32_t)a.rows * (D * 4);
}

// ---------------------------------------------------------------------------
// Attention of few query rows: up to 16 NT rows (new tokens x query heads of a
// KV head) against a sequence's pages.
//
//   work     a unit is one chunk of CR rows for each of a workgroup's four waves.
//            A launch has about as many workgroups as fit the chip, and each
//            takes one part of a (sequence, KV head) pair: `per` units, the
//            fewest with which all parts find a workgroup, by the lengths that
//            are in memory then.  The parts of a pair leave records {maximum,
//            sum, sums} and count themselves; the last to do so joins them
//            (few_join), and nothing waits.  (Equal shares that begin and end
//            inside pairs would be more even, but a workgroup's second part
//            costs its whole chain of round trips again: 32 sequences of up to
//            8,192 4-bit rows 34.5 us.)
//   loads    straight into LDS, no registers: the next chunk's keys are sent for
//            once the scores have read this one's, its values once the context
//            has; the waits count what was sent for since.  The pages of the
//            next chunks are looked up together, 64 blocks of 16 rows at a time.
//   scores   S^T = K Q^T on v_mfma_f32_16x16x32_f16: cache rows as M, the query
//            rows as N, as fp16 hi + lo images of q scale log2 e (2^-22 of it is
//            left out), two MFMAs a step, begun at minus the base.
//   softmax  lane (query n, kb) holds rows 16 t + 4 kb + v of the chunk, so e^ of
//            them stays in the lane; the base is raised only when a score passes
//            what it allows (kLift, kSlack), which spares the rescaling and the
//            exchange between lanes.
//   context  O^T = V^T P^T: the probabilities (hi + lo) are the B operand where
//            they lie, V^T comes through the transposing LDS reads (4 x 16 fp16
//            or 16 x 16 nibbles to a 16-lane group), a row of ones gives the sum.
//            Every kFold rows of a wave the sums are added to a second set, so that
//            a matrix product is never rounded to the last place of a sum that one
//            large probability or a long context has made (17 nats below one row,
//            400,000 others came out 2.8e-3 off, 6e-6 with it and kLift).
//
// Rows lie in LDS as they are, 16-byte pieces changed round within the row
// (few_turn) so that 16 rows' same piece, and the rows of a transposing read, each
// cover the banks; a load of the wave is 1 KB of consecutive rows (by pieces, 16
// bytes of each of 64 rows a load, a first chunk took twice as long).  A nibble
// becomes 64 + n in the mantissa, then one packed fma, n s - 72 s, exact as scales
// have 7 significant bits; value scales are turned into the order of the nibble
// pairs.
//
// Rows past the sequence, or of absent pages, are masked and their values
// zeroed.  fp16 rows that only some of the queries see (several new tokens) may
// hold NaN or infinity, which zero probabilities would not keep out: a chunk
// with one is added row by row.  In a chunk that all queries see nothing is looked
// for, and an image of 0 makes a NaN of an infinity: a wave whose sums are no finite
// numbers looks through its rows for what they are to be (few_odd; to look in each
// chunk instead: 64 sequences of up to 4,000 rows 72.6 us, 70.5 so).
//
// The cache's bytes bound it, the launch and a workgroup's chain of round trips
// (lengths, pages, first rows, join) where they are few: 64 sequences of up to
// 4,000 16-bit rows 70 us, 4.6 TB/s; 32 of up to 8,192 4-bit rows 31 us, 3.2 TB/s
// with some 9 us before the first and after the last row, 5.2 in between; one of
// 1,500 rows 10.8 us.
// ---------------------------------------------------------------------------
template <int D, bool Q4>
struct Few {
    static constexpr int CR = Q4 ? 64 : 32, MT = CR / 16, G = D / 32, DT = D / 16, KS = D / 32;
    static constexpr int kRow = Q4 ? D / 2 : D * 2;          // bytes
    static constexpr int kRows = CR * kRow;                  // of a chunk's keys or values
    static constexpr int PC = kRows / 1024;                  // loads of a wave for them
    static constexpr int SP = Q4 ? G / 2 : 0;                // and 4-byte pieces of a row's scales
    static constexpr int kVals = kRows, kKScale = 2 * kRows, kVScale = kKScale + SP * 256, kTurned = kVScale + SP * 256;
    static constexpr int kWave = kTurned + (Q4 ? 2 * CR * G * 2 : 0);  // values' scales s and -72 s, turned
    static constexpr int kKeyOps = PC + 2 * SP, kValOps = PC;
    static constexpr int kFold = 1024 / CR;                  // chunks of a wave between additions
    static constexpr int MS = D + 4;                         // floats of a row in the merge
    static constexpr int kMerge = 4 * 16 * MS * 4 + 4 * 16 * 8;
    static constexpr int kLds = 4 * kWave > kMerge ? 4 * kWave : kMerge;
    static_assert(kFewRows * kFewParts * 4 <= kMerge, "the parts' weights fit");
};

// Where a row keeps piece p (16 bytes).
template <int D, bool Q4>
__device__ __forceinline__ int few_turn(int row, int p) {
    if constexpr (Q4) return D == 128 ? p ^ ((row >> 2 ^ row >> 4) & 3) : p ^ ((row >> 3 ^ row >> 4) & 1);
    return D == 128 ? p ^ ((row & 7) << 1 | (row >> 3 & 1)) : p ^ ((row >> 1 & 3) << 1 | (row >> 3 & 1));
}

// lds_copy16 from an address per lane.
__device__ __forceinline__ void to_lds16(uint64_t addr, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(addr), "{m0}"(lds) : "memory");
}
// At most `n` of this wave's loads are outstanding and none of its LDS reads; no
// access moves across.
template <int n>
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4);
    asm volatile("" ::: "memory");
}

// A sequence's units (none without new tokens).
__device__ __forceinline__ int few_units(const SeqView& s, int unit) {
    return s.n > 0 ? max(1, (max(0, min(s.p0 + s.n, s.len)) + unit - 1) / unit) : 0;
}

// The S parts' records from `first` on joined by the workgroup that counted
// last.  They were written through to agent scope in this launch; the sums, whole
// cache lines that nothing here has read before, are read as usual, maximum and
// sum of a row, which share a line with other pairs', at agent scope.
template <int D, int NT>
__device__ __forceinline__ void few_join(const AttnPagedArgs& a, uint8_t* lds, const SeqView& sv, int g, int nrows, int first, int S) {
    float* const wt = reinterpret_cast<float*>(lds);  // [row][kFewParts]
    const int wave = (int)(threadIdx.x >> 6), lane = lane_id();
    const uint64_t* const ml = reinterpret_cast<const uint64_t*>(a.part + (uint64_t)(uint32_t)(a.shares * a.rows) * (D * 4));
    for (int row = wave; row < nrows; row += 4) {
        float m = -INFINITY, l = 0.0f;
        if (lane < S) {
            const uint64_t u = agent_load(ml + ((first + lane) * a.rows + row));
            m = __uint_as_float((uint32_t)u), l = __uint_as_float((uint32_t)(u >> 32));
        }
        const float M = wave_max(m);
        const float f = m == -INFINITY ? 1.0f : exp2_hw(m - M);  // no maximum: nothing seen (sums 0), or NaN only
        float L = f * l;
        for (int o = 32; o >= 1; o >>= 1) L += shfl_xor(L, o);
        if (lane < S) wt[row * kFewParts + lane] = L == 0.0f ? 0.0f : f / L;
    }
    __syncthreads();
    // all of a thread's pieces at once: their loads are what this takes
    constexpr int TR = D / 4;
    auto pieces = [&](auto number) {
        constexpr int N = decltype(number)::value;
        f32x4_t A[N];
        uint64_t from[N];
        const float* w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = (int)threadIdx.x + 256 * i, row = min(k / TR, nrows - 1);
            A[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            from[i] = a.part + (uint64_t)(uint32_t)(first * a.rows + row) * (D * 4) + 16 * (k % TR);
            w[i] = wt + row * kFewParts;
        }
#pragma unroll 8
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < N; ++i)
                A[i] += gptr<f32x4_t>(from[i] + (uint64_t)(uint32_t)(s * a.rows) * (D * 4))[0] * w[i][s];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = (int)threadIdx.x + 256 * i, row = k / TR, t = row / a.group, h = g * a.group + (row - t * a.group);
            if (row >= nrows) continue;
            const uint64_t o = a.out + ((uint64_t)(uint32_t)(sv.t0 + t) * (uint32_t)a.out_stride + (uint32_t)(h * D)) * 4;
            gptr_w<f32x4_t>(o)[k % TR] = A[i];
        }
    };
    if (nrows * TR <= 256)
        pieces(std::integral_constant<int, 1>());
    else
        pieces(std::integral_constant<int, 16 * NT * TR / 256>());
}

// The wave's columns of 16-bit values that are no finite numbers, of the rows that each
// query sees: infinities of one sign make the sum that, others NaN, and so does a row
// whose score is not finite.  Lane (n, kb) holds columns 16 d + 4 kb + u of query n.
template <int D, int NT, int DT>
__device__ __forceinline__ void few_odd(const AttnPagedArgs& a, int b, int g, int c, int r1, const int (&last)[NT], f32x4_t (&acc)[NT][DT]) {
    constexpr int CR = Few<D, false>::CR, kRow = D * 2;
    const int lane = lane_id(), kb = lane >> 4, pmask = (1 << a.c.page_log2) - 1;
    uint32_t up[NT] = {}, down[NT] = {}, nan[NT] = {};  // bit 4 d + u
    for (; c < r1; c += 4 * CR)
        for (int c16 = c; c16 < c + CR; c16 += 16) {
            const int page = c16 < r1 ? page_of(a.c, b, c16) : -1;
            if (page < 0) continue;  // the same in all lanes
            const uint64_t off = (uint64_t)(uint32_t)((c16 & pmask) * kRow);
            const uint64_t v = page_at<D, false>(a.c, a.c.v_pages, page, g) + off, k = page_at<D, false>(a.c, a.c.k_pages, page, g) + off;
            uint32_t x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
                x[r] = D == 128 ? gptr<uint32_t>(v)[r * 64 + lane] : (uint32_t)gptr<uint16_t>(v)[r * 64 + lane];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (!__ballot(odd_halves(x[r])) || c16 + r >= r1) continue;
                const uint32_t y = D == 128 ? gptr<uint32_t>(k)[r * 64 + lane] : (uint32_t)gptr<uint16_t>(k)[r * 64 + lane];
                const bool score = !__ballot(odd_halves(y));
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t e = gptr<uint16_t>(v)[r * D + 16 * d + 4 * kb + u], bit = 1u << (4 * d + u);
                        if ((e & 0x7c00u) != 0x7c00u) continue;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if (c16 + r > last[nt]) continue;
                            if (!score || (e & 0x3ffu))
                                nan[nt] |= bit;
                            else if (e & 0x8000u)
                                down[nt] |= bit;
                            else
                                up[nt] |= bit;
                        }
                    }
            }
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t bit = 1u << (4 * d + u);
                const bool p = up[nt] & bit, m = down[nt] & bit;
                if ((nan[nt] & bit) || (p && m))
                    acc[nt][d][u] = __builtin_nanf("");
                else if (p || m)
                    acc[nt][d][u] = p ? INFINITY : -INFINITY;
            }
}

// One part of a pair: units [u0, u1) of (sequence view sv, KV head g).
template <int D, bool Q4, int NT>
__device__ __forceinline__ void few_part(const AttnPagedArgs& a, uint8_t* lds, const SeqView& sv, int b, int g, int u0, int u1,
                                         bool direct) {
    using F = Few<D, Q4>;
    constexpr int CR = F::CR, MT = F::MT, G = F::G, DT = F::DT, PC = F::PC, SP = F::SP, KS = F::KS;
    const int wave = (int)(threadIdx.x >> 6), lane = lane_id(), n = lane & 15, kb = lane >> 4;
    const int nrows = sv.n * a.group;
    const int r1 = (int)min((int64_t)seen_rows(a, sv, nrows - 1), (int64_t)u1 * (4 * CR));
    LP_LDS uint8_t* const mine = (LP_LDS uint8_t*)(lds + wave * F::kWave);
    const uint32_t base = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)mine);

    // ---- loads
    const int pmask = (1 << a.c.page_log2) - 1;
    const uint32_t pbytes = (uint32_t)page_bytes(D, 1 << a.c.page_log2, Q4);
    // lane MT k + i: the page of rows 16 i .. of the wave's chunk k from c on
    auto look_up = [&](int c) {
        const int row = c + 4 * CR * (lane / MT) + 16 * (lane % MT);
        return row < r1 ? page_of(a.c, b, row) : -1;
    };
    int pages = -1, taken = 0;  // looked up, and chunks of them whose keys were sent for
    int pg = -1;                // lane: the page of block lane / (64 / MT) of the last one of these
    auto page_off = [&](int p) {
        return ((uint64_t)(uint32_t)max(p, 0) * (uint32_t)a.c.kv_heads + (uint32_t)g) * pbytes;
    };
    auto page_of_block = [&](int t) { return __builtin_amdgcn_readlane(pg, t * (64 / MT)); };
    // the wave's load p brings rows RL p .., of one or two blocks
    constexpr int RL = 1024 / F::kRow, RP = F::kRow / 16;
    auto send_rows = [&](uint64_t pool, int c, uint32_t at) {
        const uint64_t rows = pool + (Q4 ? (uint32_t)(G * 2) << a.c.page_log2 : 0u);
#pragma unroll
        for (int p = 0; p < PC; ++p) {
            const int row = lane / RP, r = RL * p + row, blk = RL * p / 16;
            const uint64_t b0 = rows + page_off(page_of_block(blk)) + (uint32_t)((c + RL * p) & pmask) * (uint32_t)F::kRow;
            uint32_t off = (uint32_t)(row * F::kRow + 16 * few_turn<D, Q4>(r, lane % RP));
            if constexpr (RL == 32) {
                // the second block's place seen from the first's (a pool may be larger than an offset)
                const uint64_t b1 = rows + page_off(page_of_block(blk + 1)) + (uint32_t)((c + RL * p + 16) & pmask) * (uint32_t)F::kRow;
                to_lds16(pick(row >= 16, b1 - 16 * F::kRow, b0) + off, at + 1024 * p);
            } else {
                lds_copy16(uniform_u64(b0), off, at + 1024 * p);
            }
        }
    };
    // 4-bit rows' scales, as they lie: row r's at 2 G r
    auto send_scales = [&](uint64_t pool, int c, uint32_t at) {
#pragma unroll
        for (int p = 0; p < SP; ++p) {
            const int r = (lane + 64 * p) / (SP ? SP : 1);  // dwords of 2 G bytes a row
            const int page = SP == 2 ? (lane & 32 ? page_of_block(2 * p + 1) : page_of_block(2 * p)) : pg;
            lds_copy4(pool + page_off(page) + (uint32_t)((c + r) & pmask) * (G * 2) + (SP == 2 ? 4 * (lane & 1) : 0), at + 256 * p);
        }
    };
    auto send_keys = [&](int c) {
        if (taken == 64 / MT) pages = look_up(c), taken = 0;
        pg = __shfl(pages, MT * taken + lane / (64 / MT), 64);
        ++taken;
        if constexpr (Q4) {
            send_scales(a.c.k_pages, c, base + F::kKScale);
            send_scales(a.c.v_pages, c, base + F::kVScale);
        }
        send_rows(a.c.k_pages, c, base);
    };
    auto send_values = [&](int c) { send_rows(a.c.v_pages, c, base + F::kVals); };
    int c = (u0 * 4 + wave) * CR;
    if (c < r1) pages = look_up(c);

    // ---- the query rows' images: lane (n, kb), step j: 8 columns, 4-bit ones in the order of nibbles8
    u32x4_t qh[NT][KS], ql[NT][KS];
    int last[NT];  // the last row that query n of a tile sees
    {
        f32x4_t x[NT][KS][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = min(nt * 16 + n, nrows - 1), i = row / a.group, h = g * a.group + (row - i * a.group);
            last[nt] = nt * 16 + n < nrows ? sv.p0 + i : -1;
            const uint64_t q = a.q + ((uint64_t)(uint32_t)(sv.t0 + i) * (uint32_t)a.q_stride + (uint32_t)(h * D)) * 4 +
                               (Q4 ? D : 32) * kb;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                x[nt][j][0] = gptr<f32x4_t>(q)[Q4 ? 2 * j : 8 * j];
                x[nt][j][1] = gptr<f32x4_t>(q)[Q4 ? 2 * j + 1 : 8 * j + 1];
            }
        }
        if (c < r1) {
            send_keys(c);
            send_values(c);
        }
        const float qs = a.scale * 1.44269504088896341f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const f32x4_t y = x[nt][j][0] * qs, z = x[nt][j][1] * qs;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if constexpr (Q4)
                        split2(y[u], z[u], hi[u], lo[u]);
                    else
                        split2(u < 2 ? y[2 * u] : z[2 * u - 4], u < 2 ? y[2 * u + 1] : z[2 * u - 3], hi[u], lo[u]);
                }
                qh[nt][j] = u32x4_t{hi[0], hi[1], hi[2], hi[3]};
                ql[nt][j] = u32x4_t{lo[0], lo[1], lo[2], lo[3]};
            }
    }
    const int all = seen_rows(a, sv, 0);  // rows below it are seen by every query row

    float m[NT];  // the base, -inf before the first score
    f32x4_t acc[NT][DT], sum[NT];
    f32x4_t acc2[NT][DT];  // and what was put aside
    float sum2[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY, sum[nt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, sum2[nt] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[nt][d] = sum[nt], acc2[nt][d] = sum[nt];
    }
    auto fold = [&] {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            sum2[nt] += sum[nt][0], sum[nt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DT; ++d) acc2[nt][d] += acc[nt][d], acc[nt][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    int until_fold = 1;  // (a context's first row is often the large one)
    bool odd_may = false;
    for (; c < r1; c += 4 * CR) {
        wait_loads<F::kValOps>();  // the keys (and scales) are here
        // a bit per block of 16 rows: its page is there
        const uint64_t pages_in = __ballot(pg >= 0);
        uint32_t there = 0;
#pragma unroll
        for (int t = 0; t < MT; ++t) there |= (uint32_t)(pages_in >> (t * (64 / MT)) & 1) << t;
        const bool whole = c + CR <= all && there == (1u << MT) - 1;  // all there and seen by all
        if constexpr (Q4) {
            // the value scales by group, in the order of the pairs of rows (t even, t
            // odd) that a lane group multiplies; of rows that are not there 0
            const bool in = pg >= 0 && c + lane < r1;
            const int at = 16 * (lane >> 2 & 3) + 8 * (kb >> 1) + 2 * (lane & 3) + (kb & 1);
            uint32_t v[SP];
            if constexpr (SP == 2) {
                const uint64_t x = *(LP_LDS u64_any*)(mine + F::kVScale + 8 * lane);
                v[0] = (uint32_t)x, v[1] = (uint32_t)(x >> 32);
            } else {
                v[0] = *(LP_LDS u32_any*)(mine + F::kVScale + 4 * lane);
            }
#pragma unroll
            for (int p = 0; p < SP; ++p) {
                v[p] = in ? v[p] : 0u;
                const half2_t y = __builtin_bit_cast(half2_t, v[p]) * (_Float16)-72.0f;
                const uint32_t w = __builtin_bit_cast(uint32_t, y);
                LP_LDS u16_any* const t = (LP_LDS u16_any*)(mine + F::kTurned) + 4 * p * CR + at;
                t[0] = (uint16_t)v[p], t[2 * CR] = (uint16_t)(v[p] >> 16);
                t[CR] = (uint16_t)w, t[3 * CR] = (uint16_t)(w >> 16);
            }
        }
        // ---- scores
        f32x4_t s[NT][MT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float from = m[nt] == -INFINITY ? 0.0f : -m[nt];
#pragma unroll
            for (int t = 0; t < MT; ++t) s[nt][t] = f32x4_t{from, from, from, from};
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            u32x4_t k[KS];
            if constexpr (Q4) {
                const int r = 16 * t + n;
                const uint16_t sx = *(LP_LDS u16_any*)(mine + F::kKScale + r * (G * 2) + 2 * (kb * G >> 2));  // the lane's columns' group
                const _Float16 x = __builtin_bit_cast(_Float16, sx);
                const half2_t x2 = {x, x}, y2 = x2 * (_Float16)-72.0f;
                const half2_t sc[4] = {x2, x2, x2, x2}, cc[4] = {y2, y2, y2, y2};
                if constexpr (D == 128) {
                    const u32x4_t w = *(LP_LDS u32x4_any*)(mine + r * F::kRow + 16 * few_turn<D, Q4>(r, kb));
#pragma unroll
                    for (int j = 0; j < KS; ++j) k[j] = nibbles8(w[j], sc, cc);
                } else {
                    const uint64_t w = *(LP_LDS u64_any*)(mine + r * F::kRow + 16 * few_turn<D, Q4>(r, kb >> 1) + 8 * (kb & 1));
                    k[0] = nibbles8((uint32_t)w, sc, cc);
                    k[1] = nibbles8((uint32_t)(w >> 32), sc, cc);
                }
            } else {
#pragma unroll
                for (int j = 0; j < KS; ++j)
                    k[j] = *(LP_LDS u32x4_any*)(mine + (16 * t + n) * F::kRow + 16 * few_turn<D, Q4>(n, 4 * j + kb));
            }
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][t] = mfma16(k[j], qh[nt][j], s[nt][t]);
                    s[nt][t] = mfma16(k[j], ql[nt][j], s[nt][t]);
                }
        }
        const bool more = c + 4 * CR < r1;
        if (more) {
            wait_loads<63>();  // the keys and scales are read
            send_keys(c + 4 * CR);
        }
        // ---- softmax: lane (n, kb), row 16 t + 4 kb + v
        u32x4_t ph[NT][CR / 32], pl[NT][CR / 32];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (!whole) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (!(there >> t & 1) || c + 16 * t + 4 * kb + v > last[nt]) s[nt][t][v] = -INFINITY;
            }
            float mx = s[nt][0][0];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[nt][t][v]);
            if (__ballot(mx > (m[nt] == -INFINITY ? -INFINITY : kLift + kSlack))) {
                mx = fmaxf(mx, shfl_xor(mx, 16));
                mx = fmaxf(mx, shfl_xor(mx, 32));
                const bool first = m[nt] == -INFINITY;
                const float by = first ? (mx == -INFINITY ? 0.0f : mx - kLift) : fmaxf(mx - kLift, 0.0f);
                const float f = first ? 0.0f : exp2_hw(-by);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v) s[nt][t][v] -= by;
                sum[nt] *= f, sum2[nt] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[nt][d] *= f, acc2[nt][d] *= f;
                m[nt] = first ? mx - kLift : m[nt] + by;
            }
#pragma unroll
            for (int w = 0; w < CR / 32; ++w)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint32_t hi, lo;
                    if constexpr (Q4)
                        split2(exp2_hw(s[nt][2 * w][v]), exp2_hw(s[nt][2 * w + 1][v]), hi, lo);
                    else
                        split2(exp2_hw(s[nt][v >> 1][2 * (v & 1)]), exp2_hw(s[nt][v >> 1][2 * (v & 1) + 1]), hi, lo);
                    ph[nt][w][v] = hi, pl[nt][w][v] = lo;
                }
        }
        // ---- context
        if (more)
            wait_loads<F::kKeyOps>();  // the values are here
        else
            wait_loads<0>();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int w = 0; w < CR / 32; ++w) {
                const u32x4_t one = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
                sum[nt] = mfma16(one, ph[nt][w], sum[nt]);
                sum[nt] = mfma16(one, pl[nt][w], sum[nt]);
            }
        bool apart = false;
        if constexpr (!Q4) {
            if (!whole) {
                // rows that are not there: zeros; an odd value among the others
                bool odd = false;
                for (int i = lane; i < F::kRows / 16; i += 64) {
                    const int r = i / (F::kRow / 16);
                    LP_LDS u32x4_any* const at = (LP_LDS u32x4_any*)(mine + F::kVals + 16 * i);
                    u32x4_t x = *at;
                    const bool in = (there >> (r >> 4) & 1) && c + r < r1;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        x[u] = in ? x[u] : 0u;
                        odd |= odd_halves(x[u]);
                    }
                    *at = x;
                }
                apart = __ballot(odd) != 0;
                __builtin_amdgcn_wave_barrier();
            }
        }
        odd_may |= whole || apart;
        if (apart) {
            // row by row, each for the queries that see it
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int t = e / 4, v = e % 4;  // its probability: half e % 2 of word e / 2
                    const half2_t hi = __builtin_bit_cast(half2_t, (uint32_t)ph[nt][0][e / 2]), lo = __builtin_bit_cast(half2_t, (uint32_t)pl[nt][0][e / 2]);
                    const float p = (float)hi[e % 2] + (float)lo[e % 2];
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        const int r = 16 * t + 4 * k + v;
                        const float pk = __shfl(p, n + 16 * k, 64);
                        if (c + r > last[nt] || !(there >> t & 1)) continue;
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const int dim = 16 * d + 4 * kb + u;
                                const uint32_t x = *(LP_LDS u16_any*)(mine + F::kVals + r * F::kRow + 16 * few_turn<D, Q4>(r, dim / 8) + 2 * (dim % 8));
                                acc[nt][d][u] = __builtin_fmaf(pk, f16_bits_to_f32(x), acc[nt][d][u]);
                            }
                    }
                }
        } else if constexpr (Q4) {
            const int vr = 16 * (n >> 2) + 4 * kb + (n & 3);
#pragma unroll
            for (int u = 0; u < G; ++u) {
                half2_t sc[2][4], cc[2][4];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    LP_LDS u16_any* const at = (LP_LDS u16_any*)(mine + F::kTurned) + 2 * u * CR + 16 * kb + 8 * w;
                    const u32x4_t x = *(LP_LDS u32x4_any*)at, y = *(LP_LDS u32x4_any*)(at + CR);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t xi = x[i], yi = y[i];  // (a bit cast of the element itself reads element 0)
                        sc[w][i] = __builtin_bit_cast(half2_t, xi), cc[w][i] = __builtin_bit_cast(half2_t, yi);
                    }
                }
                v2i32_t x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    x[e] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((LP_LDS v2i32_t*)(uintptr_t)(base + F::kVals + (uint32_t)(vr * F::kRow + 16 * few_turn<D, Q4>(vr, u) + 8 * e)));
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const u32x4_t v = nibbles8((uint32_t)x[e][w], sc[w], cc[w]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            acc[nt][2 * u + e] = mfma16(v, ph[nt][w], acc[nt][2 * u + e]);
                            acc[nt][2 * u + e] = mfma16(v, pl[nt][w], acc[nt][2 * u + e]);
                        }
                    }
            }
        } else {
            const int vr = 4 * kb + (n >> 2);  // and 16 rows further
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint32_t at = base + F::kVals + (uint32_t)(vr * F::kRow + 16 * few_turn<D, Q4>(vr, 2 * d + (n >> 1 & 1)) + 8 * (n & 1));
                const v4i16_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP_LDS v4i16_t*)(uintptr_t)at);
                const v4i16_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP_LDS v4i16_t*)(uintptr_t)(at + 16 * F::kRow));
                const v2i32_t y0 = __builtin_bit_cast(v2i32_t, x0), y1 = __builtin_bit_cast(v2i32_t, x1);
                const u32x4_t v = {(uint32_t)y0[0], (uint32_t)y0[1], (uint32_t)y1[0], (uint32_t)y1[1]};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    acc[nt][d] = mfma16(v, ph[nt][0], acc[nt][d]);
                    acc[nt][d] = mfma16(v, pl[nt][0], acc[nt][d]);
                }
            }
        }
        if (more) {
            wait_loads<63>();  // the values are read
            send_values(c + 4 * CR);
        }
        if (more && --until_fold == 0) fold(), until_fold = F::kFold;
    }
    fold();
    if (!Q4 && odd_may) {
        f32x4_t odd = {0.0f, 0.0f, 0.0f, 0.0f};  // or NaN
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int u = 0; u < 4; ++u) odd[u] = __builtin_fmaf(acc2[nt][d][u], 0.0f, odd[u]);
        if (__builtin_expect(__ballot(!(odd[0] + odd[1] + odd[2] + odd[3] == 0.0f)) != 0, 0)) few_odd<D, NT, DT>(a, b, g, (u0 * 4 + wave) * CR, r1, last, acc2);
    }

    // ---- the waves' sums meet, a query tile at a time: the output, or the part's record
    constexpr int MS = F::MS;
    float* const sums = reinterpret_cast<float*>(lds);  // [wave][n][MS]
    float2_any* const ml = reinterpret_cast<float2_any*>(lds + 4 * 16 * MS * 4);
    const uint64_t rml = a.part + (uint64_t)(uint32_t)(a.shares * a.rows) * (D * 4);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_any*>(sums + (wave * 16 + n) * MS + 16 * d + 4 * kb) = acc2[nt][d];
        if (kb == 0) ml[wave * 16 + n] = make_float2(m[nt], sum2[nt]);
        __syncthreads();
        constexpr int TR = D / 4;  // threads of a row
#pragma unroll
        for (int k = 0; k < 16 * TR; k += 256) {
            const int q = (k + (int)threadIdx.x) / TR, d4 = (k + (int)threadIdx.x) % TR, row = nt * 16 + q;
            if (row >= nrows) continue;
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w * 16 + q].x);
            f32x4_t A = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float2 x = ml[w * 16 + q];
                const float f = x.x == -INFINITY ? 1.0f : exp2_hw(x.x - M);  // as in few_join
                L = __builtin_fmaf(f, x.y, L);
                A += *reinterpret_cast<const f32x4_any*>(sums + (w * 16 + q) * MS + 4 * d4) * f;
            }
            if (direct) {
                const int i = row / a.group, h = g * a.group + (row - i * a.group);
                const uint64_t o = a.out + ((uint64_t)(uint32_t)(sv.t0 + i) * (uint32_t)a.out_stride + (uint32_t)(h * D)) * 4;
                const float f = L == 0.0f ? 0.0f : 1.0f / L;
                gptr_w<f32x4_t>(o)[d4] = A * f;
            } else {
                const uint32_t at = blockIdx.x * (uint32_t)a.rows + (uint32_t)row;
                uint64_t* const o = reinterpret_cast<uint64_t*>(a.part + (uint64_t)at * (D * 4) + 16 * d4);
                const float a0 = A[0], a1 = A[1], a2 = A[2], a3 = A[3];
                agent_store(o, (uint64_t)__float_as_uint(a1) << 32 | __float_as_uint(a0));
                agent_store(o + 1, (uint64_t)__float_as_uint(a3) << 32 | __float_as_uint(a2));
                if (d4 == 0)
                    agent_store(reinterpret_cast<uint64_t*>(rml) + at, (uint64_t)__float_as_uint(L) << 32 | __float_as_uint(M));
            }
        }
    }
}

template <int D, bool Q4, int NT>
__device__ __forceinline__ void few_body(const AttnPagedArgs& a) {
    using F = Few<D, Q4>;
    constexpr int kUnit = 4 * F::CR;
    __shared__ __align__(1024) uint8_t lds[F::kLds];
    __shared__ int flag;
    const int lane = lane_id(), kv = a.c.kv_heads;
    int b, g, part = 0, parts = 1, per = INT32_MAX / kUnit;
    SeqView sv{0, 0, 0, 0};
    if (a.shares) {
        // units in a lane each (64 sequences), or in LDS
        int* const many = reinterpret_cast<int*>(lds);
        const bool lanes = a.batch <= 64;
        int mine = 0, total = 0;
        if (lanes) {
            if (lane < a.batch) sv = seq_view(a, lane);
            mine = few_units(sv, kUnit);
            total = __builtin_amdgcn_readlane(wave_incl_scan(mine), 63);
        } else {
            for (int i = threadIdx.x; i < (a.batch + 63 & ~63); i += 256)
                many[i] = i < a.batch ? few_units(seq_view(a, i), kUnit) : 0;
            __syncthreads();
            for (int i = 0; i < a.batch; i += 64) total += __builtin_amdgcn_readlane(wave_incl_scan(many[i + lane]), 63);
        }
        auto parts_of = [&](int u) { return (u + per - 1) / per; };
        per = max((total * kv + a.shares - 1) / a.shares, a.min_units);
        for (;; per += (per + 7) / 8) {
            int n = 0;
            for (int i = 0; i < a.batch; i += 64) n += __builtin_amdgcn_readlane(wave_incl_scan(parts_of(lanes ? mine : many[i + lane])), 63);
            if (n * kv <= a.shares) break;  // one part a pair always fits
        }
        // the sequence whose parts hold the workgroup's number
        int before = 0, at = (int)blockIdx.x;
        for (b = 0;; b += 64) {
            if (b >= a.batch) return;  // whole workgroups, here and below
            const int n = parts_of(lanes ? mine : many[b + lane]), incl = before + kv * wave_incl_scan(n);
            const int i = __popcll(__ballot(incl <= at));
            if (i < 64) {
                parts = __builtin_amdgcn_readlane(n, i);
                at -= __builtin_amdgcn_readlane(incl, i) - kv * parts;
                b += i;
                break;
            }
            before = __builtin_amdgcn_readlane(incl, 63);
        }
        g = at / parts, part = at - g * parts;
        if (lanes) {
            sv = SeqView{__builtin_amdgcn_readlane(sv.t0, b), __builtin_amdgcn_readlane(sv.n, b),
                         __builtin_amdgcn_readlane(sv.len, b), __builtin_amdgcn_readlane(sv.p0, b)};
        } else {
            sv = seq_view(a, b);
            __syncthreads();  // the LDS is free
        }
    } else {  // a workgroup per pair
        b = (int)blockIdx.x / kv, g = (int)blockIdx.x - b * kv;
        sv = seq_view(a, b);
        if (sv.n <= 0) return;
    }
    few_part<D, Q4, NT>(a, lds, sv, b, g, part * per, part * per + per, parts == 1);
    if (parts == 1) return;
    int* const count = reinterpret_cast<int*>(a.sync) + (b * kv + g) * kPagedStride;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        const int o = atomicAdd(count, 1);
        if (o == parts - 1) agent_store(count, 0);  // the last: zero for the next launch
        flag = o;
    }
    __syncthreads();
    if (flag == parts - 1) few_join<D, NT>(a, lds, sv, g, sv.n * a.group, (int)blockIdx.x - part, parts);
}

}  // namespace

// (waves a SIMD that the registers leave room for; with 4-bit rows of 128 the second set
// of sums takes the third: 256 sequences' 4 KV heads over up to 2,000 rows 67 us, 62 with
// three and one set, 95 with three and both, spilled)
#define LP_ATTN_FEW(NAME, WAVES, D, Q4, NT) \
    extern "C" __global__ void __launch_bounds__(256, WAVES) lp_attn_few_##NAME(const AttnPagedArgs a) { few_body<D, Q4, NT>(a); }
LP_ATTN_FEW(f16_d64, 2, 64, false, 1)
LP_ATTN_FEW(f16_d128, 2, 128, false, 1)
LP_ATTN_FEW(q4_d64, 3, 64, true, 1)
LP_ATTN_FEW(q4_d128, 2, 128, true, 1)
LP_ATTN_FEW(f16_d64_n2, 2, 64, false, 2)
LP_ATTN_FEW(f16_d128_n2, 1, 128, false, 2)
LP_ATTN_FEW(q4_d64_n2, 2, 64, true, 2)
LP_ATTN_FEW(q4_d128_n2, 1, 128, true, 2)
#undef LP_ATTN_FEW

// ---------------------------------------------------------------------------
// Attention of many query rows: a workgroup takes 128 of a (sequence, KV head)'s
// query rows, 32 a wave, and walks the rows of the context that they see in
// chunks of 64, as fp16 in LDS for its four waves, one barrier a chunk: the next
// chunk's rows are written there (4-bit ones multiplied out on the way, columns of
// eight in the order of nibbles8) and the one's after it sent for while this one is
// worked on.
//
// Matrix work bounds it: fp32 queries and probabilities cost two fp16 MFMAs a
// product.  As above S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_32x32x16_f16: the
// queries' images stay in registers, the probabilities are the B operand where
// they lie (lane (query n, h), value r: row 8 (r / 4) + 4 h + r % 4 of 32), V^T
// comes through transposing reads of 4 x 16 blocks, and a row read from LDS
// serves the hi and the lo product.  Key rows are padded by 16 bytes (16 rows'
// 16-byte pieces then cover the banks), value rows by 64 (four rows' 32 bytes and
// their neighbours' do).  The order of the instructions is given: every two MFMAs
// have the reads for those two steps on and a share of the vector work beside them
// (left to the compiler, each pair waited for its own reads: 526 us against 432).
// What would hold the accumulators twice, a branch that computes them in another
// way, stays out of the loop.
//
// fp32 sums that hold one large probability are rounded to the last place of it at
// each step of a matrix product, so that thousands of small ones behind it come out
// wrong together, the low images' products first.  Every kLook chunks (and after the
// first, the second and the fourth) a wave compares what they added with the sum so far;
// where a query row's is, for each chunk, below kFaint of that, the accumulators are put
// aside in memory, where the result goes, and begin again (one row 17 nats above
// 100,000: 6.4e-3 off without this and kLift, 9e-6 with them; at worst, every time that
// a wave looks, 2,048 tokens behind 6,001 rows take 440 us instead of 410).
//
// 2,048 tokens of 32 heads on 4 KV heads behind 6,001 rows of 16 bits: 407 to 418
// us, 565 to 580 TFLOP/s of the formula's and twice that of MFMA work, what a large fp16 product
// reaches; 12 sequences of up to 5 tokens, 16 heads to a KV head, behind up to
// 6,000 rows of 4 bits: 35 us, of which a chunk takes about 2.8 us (the steps' vector
// work, a wave's alone) and the launch with what comes before the first one 10; six
// prompts of up to 700 tokens, 32 heads on 4: 53 us, the longest one's last tiles.
// (Pages looked at as soon as asked for: 424 us, the prompts of one length 87
// against 81.)
// ---------------------------------------------------------------------------
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16_t mfma32(const u32x4_t& a, const u32x4_t& b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

constexpr int kLook = 8;  // chunks
constexpr float kFaint = 0x1p-8f;

template <int D>
struct ManyRows {
    static constexpr int CR = 64;
    static constexpr int RSK = D * 2 + 16, RSV = D * 2 + 64;
    static constexpr int kBuf = CR * (RSK + RSV);
    static constexpr int kFlags = 2 * kBuf;  // 4 waves' ballots of rows there per buffer, 4 words of odd values
    static constexpr int kAside = kFlags + 2 * 4 * 8 + 4 * 4;  // a thread's sum put aside, with its base
    static constexpr int kLds = kAside + 256 * 8;
};

template <int D, bool Q4>
__device__ __forceinline__ void many_body(const AttnPagedArgs& a) {
    using M = ManyRows<D>;
    constexpr int CR = M::CR, RSK = M::RSK, RSV = M::RSV, G = D / 32;
    constexpr int KS = D / 16, DT = D / 32;
    constexpr int W = Q4 ? D / 32 : D / 8;  // 32-bit words of a row's quarter
    __shared__ __align__(16) uint8_t lds[M::kLds];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = lane_id(), n = lane & 31, h = lane >> 5;
    // The longest first: the last tiles of all pairs, then those before them (pair
    // by pair, each kept to an XCD: ragged prompts 75.6 us against 61.7), and the
    // last spans, which may be short, behind the others.  Each time round the pairs
    // are shifted by one, so that a pair's workgroups are shared among the XCDs, to
    // which consecutive ones go in turn (two sequences of 4 KV heads, 4,096 and about
    // half as many tokens: 705 us without, 464 with it).  Where all are on the card
    // at once, two a CU, the second ones go from the shortest up (426 us, 419).
    const int pairs = a.batch * a.c.kv_heads, total = pairs * a.tiles;
    int id = (int)blockIdx.x % total;
    const int split = (int)blockIdx.x / total;
    if (id >= 256 && total <= 512) id = total - 1 - (id - 256);
    const int bg = (id + id / pairs + split) % pairs, tile = a.tiles - 1 - id / pairs;
    const int b = bg / a.c.kv_heads, g = bg - b * a.c.kv_heads;
    const SeqView sv = seq_view(a, b);
    const int nrows = sv.n * a.group, row0 = tile * kManyRows;
    if (row0 >= nrows) return;  // whole workgroups, here and below
    const int vis = seen_rows(a, sv, min(row0 + kManyRows, nrows) - 1);
    const int r0 = split * a.span, r1 = min(vis, r0 + a.span);
    if (r0 >= r1 && split > 0) return;
    const uint32_t lbase = (uint32_t)(uintptr_t)(LP_LDS uint8_t*)lds;
    LP_LDS uint8_t* const ll = (LP_LDS uint8_t*)lds;

    // ---- staging: thread (row tid / 4, quarter tid % 4) of a chunk
    const int srow = tid >> 2, quarter = tid & 3;
    const int pmask = (1 << a.c.page_log2) - 1;

    uint32_t kreg[W], vreg[W];
    uint32_t ks = 0, vs = 0;
    // a row's page, asked for and, later, looked at: what asks waits for nothing
    auto ask_page = [&](int c) {  // (r1 is within the table's width)
        const uint32_t col = (uint32_t)(min(c + srow, r1 - 1) >> a.c.page_log2);
        return gptr<int>(a.c.table)[(uint64_t)(uint32_t)b * (uint32_t)a.c.max_pages + col];
    };
    auto page_for = [&](int asked, int c) {
        asm volatile("" : "+v"(asked));
        return c + srow < r1 && (uint32_t)asked < (uint32_t)a.c.pages ? asked : -1;
    };
    auto load_rows = [&](uint32_t (&r)[W], uint32_t& s, uint64_t pool, int c, int pg) {
        const uint32_t pr = (uint32_t)((c + srow) & pmask);
        const uint64_t at = page_at<D, Q4>(a.c, pool, max(pg, 0), g);
        if constexpr (Q4) {
            s = gptr<uint16_t>(at)[pr * G + (quarter * G >> 2)];
            const uint64_t ra = at + ((uint32_t)(G * 2) << a.c.page_log2) + pr * (D / 2) + quarter * (D / 8);
            if constexpr (D == 64) {
                const uint64_t v = *gptr<uint64_t>(ra);
                r[0] = (uint32_t)v, r[1] = (uint32_t)(v >> 32);
            } else {
                const u32x4_t v = *gptr<u32x4_t>(ra);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < W / 4; ++j) {
                const u32x4_t v = *gptr<u32x4_t>(at + pr * (D * 2) + 16 * quarter + 64 * j);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[4 * j + i] = v[i];
            }
        }
    };
    using Finite = std::false_type;
    using Odd = std::true_type;
    // ODD: only what is no finite number of the values; else that is left out, and
    // `strange` says that there was some.  The values of rows that are not there are 0.
    int strange = 0;
    // (16-bit ones: whether a wave's rows under way need that, and it done)
    auto special = [&](int c, int pg) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < W; ++i)
            most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, most),
                                                                          __builtin_bit_cast(u16x2_t, vreg[i] & 0x7fff7fffu)));
        return __ballot(odd_halves(most) || c + srow >= r1 || pg < 0) != 0;
    };
    auto mend = [&](auto odd_pass, int c, int pg) {
        constexpr bool ODD = decltype(odd_pass)::value;
        const bool in = c + srow < r1 && pg >= 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const uint32_t lo = in ? vreg[i] & 0xffffu : 0u, hi = in ? vreg[i] & 0xffff0000u : 0u;
            strange |= odd_halves(lo) || odd_halves(hi);
            vreg[i] = (odd_halves(lo) == ODD ? lo : 0u) | (odd_halves(hi) == ODD ? hi : 0u);
        }
    };
    // a chunk to LDS, in KS pieces
    struct Scales {
        half2_t s[4], c[4];
    } ksc, vsc;
    auto store_begin = [&](auto odd_pass, int buf, int c, int pg) {
        constexpr bool ODD = decltype(odd_pass)::value;
        const bool in = c + srow < r1 && pg >= 0;
        if constexpr (Q4) {
            const uint32_t ke = in ? ks | ks << 16 : 0u;
            uint32_t ve = in ? vs | vs << 16 : 0u;
            const bool odd = odd_halves(ve);
            strange |= odd;
            ve = odd == ODD ? ve : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ksc.s[i] = __builtin_bit_cast(half2_t, ke), ksc.c[i] = ksc.s[i] * (_Float16)-72.0f;
                vsc.s[i] = __builtin_bit_cast(half2_t, ve), vsc.c[i] = vsc.s[i] * (_Float16)-72.0f;
            }
        }
        *(LP_LDS u64_any*)(ll + M::kFlags + buf * 32 + wave * 8) = __ballot(in);  // one word, from all lanes
    };
    auto store_piece = [&](int buf, int j) {
        const int i = j >> 1;
        const uint32_t at = (uint32_t)(buf * M::kBuf + (j & 1 ? CR * RSK + srow * RSV : srow * RSK));
        if constexpr (Q4)
            *(LP_LDS u32x4_any*)(ll + at + quarter * (16 * W) + 16 * i) =
                j & 1 ? nibbles8(vreg[i], vsc.s, vsc.c) : nibbles8(kreg[i], ksc.s, ksc.c);
        else
            *(LP_LDS u32x4_any*)(ll + at + 16 * quarter + 64 * i) =
                j & 1 ? u32x4_t{vreg[4 * i], vreg[4 * i + 1], vreg[4 * i + 2], vreg[4 * i + 3]}
                      : u32x4_t{kreg[4 * i], kreg[4 * i + 1], kreg[4 * i + 2], kreg[4 * i + 3]};
    };
    auto store_rows = [&](auto odd_pass, int buf, int c, int pg) {
        store_begin(odd_pass, buf, c, pg);
#pragma unroll
        for (int j = 0; j < KS; ++j) store_piece(buf, j);
    };
    int pg = -1, pg1 = -1;  // of the chunk in the registers, and of the one after it
    if (r0 < r1) {
        pg = ask_page(r0);
        const int next = ask_page(r0 + CR);
        pg = page_for(pg, r0);
        load_rows(kreg, ks, a.c.k_pages, r0, pg);
        load_rows(vreg, vs, a.c.v_pages, r0, pg);
        pg1 = page_for(next, r0 + CR);
    }

    // ---- the wave's query rows
    const int row = row0 + 32 * wave + n, qi = row / a.group, qh_ = g * a.group + (row - qi * a.group);
    const bool on = row < nrows;
    const int last = on ? sv.p0 + qi : -1;
    const int wrow = min(row0 + 32 * wave + 31, nrows - 1);
    const int wvis = row0 + 32 * wave < nrows ? seen_rows(a, sv, wrow) : 0;        // rows that one of the wave's sees
    const int wall = row0 + 32 * wave < nrows ? seen_rows(a, sv, row0 + 32 * wave) : 0;  // rows that all of them see
    u32x4_t qh[KS], ql[KS];
    {
        const float qs = a.scale * 1.44269504088896341f;
        const uint64_t q = a.q + ((uint64_t)(uint32_t)(sv.t0 + (on ? qi : 0)) * (uint32_t)a.q_stride + (uint32_t)((on ? qh_ : 0) * D)) * 4;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            f32x4_t x0 = gptr<f32x4_t>(q + 64 * j + 32 * h)[0], x1 = gptr<f32x4_t>(q + 64 * j + 32 * h)[1];
#pragma unroll
            for (int u = 0; u < 4; ++u) x0[u] = on ? x0[u] * qs : 0.0f, x1[u] = on ? x1[u] * qs : 0.0f;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (Q4)
                    split2(x0[u], x1[u], hi[u], lo[u]);
                else
                    split2(u < 2 ? x0[2 * u] : x1[2 * u - 4], u < 2 ? x0[2 * u + 1] : x1[2 * u - 3], hi[u], lo[u]);
            }
            qh[j] = u32x4_t{hi[0], hi[1], hi[2], hi[3]};
            ql[j] = u32x4_t{lo[0], lo[1], lo[2], lo[3]};
        }
    }
    // the lane's places in a chunk: a key row's piece, and its share of 4 x 16 values
    // (behind the asm so that what is added to them stays in the reads' offsets)
    uint32_t klane = lbase + (uint32_t)(n * RSK + 16 * h);
    uint32_t vlane = lbase + (uint32_t)(CR * RSK + (4 * h + (lane >> 2 & 3)) * RSV + 32 * (lane >> 4 & 1) + 8 * (lane & 3));
    asm volatile("" : "+v"(klane), "+v"(vlane));
    // the base, the lane's sum since the last look at it, and what went before that and is
    // in the accumulators
    float m = -INFINITY, l = 0.0f, lseg = 0.0f;
    // (in LDS, for the loop has no register left) the sum of what was put aside, with its base
    LP_LDS f32_any* const aside = (LP_LDS f32_any*)(ll + M::kAside + tid * 8);
    bool put = false;
    f32x16_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;

    auto load_next = [&](int c) {  // (rows behind the last are some page's)
        pg = pg1;
        load_rows(kreg, ks, a.c.k_pages, c, pg);
        load_rows(vreg, vs, a.c.v_pages, c, pg);
    };
    const bool none = r0 >= r1;
    if (!none) {
        if (!Q4 && special(r0, pg)) mend(Finite(), r0, pg);
        store_rows(Finite(), 0, r0, pg);
        const int next = ask_page(r0 + 2 * CR);
        load_next(r0 + CR);
        if (!Q4 && special(r0 + CR, pg)) mend(Finite(), r0 + CR, pg);
        pg1 = page_for(next, r0 + 2 * CR);
        __syncthreads();
    }
    int buf = 0;
    auto keys = [&](int t, int j) {
        return *(LP_LDS u32x4_any*)(uintptr_t)(klane + (uint32_t)(buf * M::kBuf + 32 * t * RSK + 32 * j));
    };
    auto values = [&](int i) {  // rows 16 (i / DT).., columns 32 (i % DT)..
        const uint32_t at = vlane + (uint32_t)(buf * M::kBuf + 16 * (i / DT) * RSV + 64 * (i % DT));
        const v2i32_t x = __builtin_bit_cast(v2i32_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP_LDS v4i16_t*)(uintptr_t)at));
        const v2i32_t y = __builtin_bit_cast(v2i32_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP_LDS v4i16_t*)(uintptr_t)(at + 8 * RSV)));
        return u32x4_t{(uint32_t)x[0], (uint32_t)x[1], (uint32_t)y[0], (uint32_t)y[1]};
    };
    auto zero = [] {
        f32x16_t s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
        return s;
    };
    // what rows c + 32 t.. hold no value for, and what the query does not see
    auto mask = [&](int c, int t, f32x16_t& s) {
        int h4 = 4 * h;  // behind the asm so that nothing of this is kept in registers meanwhile
        asm volatile("" : "+v"(h4));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t there = *(LP_LDS u64_any*)(ll + M::kFlags + buf * 32 + (2 * t + i) * 8);  // four bits a row
#pragma unroll
            for (int r = 8 * i; r < 8 * i + 8; ++r) {
                const int rr = 8 * (r / 4) + h4 + r % 4;
                if (!(there >> (4 * (rr & 15)) & 1) || c + 32 * t + rr > last) s[r] = -INFINITY;
            }
        }
    };
    auto top = [&](const f32x16_t& s) {
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        return mx;
    };
    // to a larger base; what the sums so far are to be multiplied by
    auto raise = [&](float mx) {
        mx = fmaxf(mx, shfl_xor(mx, 32)) - kLift;
        const float mn = fmaxf(m, mx);
        const float f = m == -INFINITY ? 0.0f : exp2_hw(m - mn);
        l *= f, lseg *= f;
        m = mn;
        return f;
    };
    auto scale = [&](float f) {
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= f;
    };
    // the lane's part of the query row's output or record: columns 32 d + 8 e .., 4-bit
    // ones' place 4 h + r of eight column (4 h + r) / 2 + 4 (r % 2)
    struct Place {
        uint64_t at, rec;
        int h;
        bool on, direct;
    };
    auto place = [&] {
        int me = lane;  // behind the asm so that nothing of this is kept in registers meanwhile
        asm volatile("" : "+v"(me));
        Place p;
        const int r = row0 + 32 * wave + (me & 31), t = r / a.group, head = g * a.group + (r - t * a.group);
        p.h = me >> 5, p.on = r < nrows, p.direct = vis <= a.span;
        p.rec = rec_index(a, bg, split, r);
        p.at = p.direct ? a.out + ((uint64_t)(uint32_t)(sv.t0 + t) * (uint32_t)a.out_stride + (uint32_t)(head * D)) * 4
                        : a.part + p.rec * (D * 4);
        return p;
    };
    auto get4 = [&](const Place& p, int d, int e) {
        if constexpr (Q4) {
            const uint64_t o = p.at + (32 * d + 8 * e + 2 * p.h) * 4;
            const float2 x = gptr<float2>(o)[0], y = gptr<float2>(o)[2];
            return f32x4_t{x.x, y.x, x.y, y.y};
        } else {
            return gptr<f32x4_t>(p.at + (32 * d + 8 * e + 4 * p.h) * 4)[0];
        }
    };
    auto put4 = [&](const Place& p, int d, int e, const f32x4_t& x) {
        if constexpr (Q4) {
            const uint64_t o = p.at + (32 * d + 8 * e + 2 * p.h) * 4;
            gptr_w<float2>(o)[0] = make_float2(x[0], x[2]);
            gptr_w<float2>(o)[2] = make_float2(x[1], x[3]);
        } else {
            gptr_w<f32x4_t>(p.at + (32 * d + 8 * e + 4 * p.h) * 4)[0] = x;
        }
    };
    auto part4 = [&](int d, int e) {
        return f32x4_t{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
    };
    // the sum that was put aside, and what goes with it is to be multiplied by (no base:
    // it is 0, or a NaN that stays)
    auto sum_aside = [&](float& f) {
        const float x = aside[0], from = aside[1];
        f = from == -INFINITY ? 1.0f : exp2_hw(from - m);
        return x * f;
    };
    // what `chunks` chunks have added since the last time against what the accumulators hold
    auto look = [&](int chunks) {
        const bool faint = __ballot(l > 0.0f && l < lseg * (kFaint * (float)chunks)) != 0;
        lseg += l, l = 0.0f;
        if (!faint) return;
        float f = 1.0f, sum = 0.0f;
        if (put) sum = sum_aside(f);
        const Place p = place();
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (p.on) {
                    f32x4_t x = part4(d, e);
                    if (put) x += get4(p, d, e) * f;
                    put4(p, d, e, x);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[d][4 * e + u] = 0.0f;
                __builtin_amdgcn_sched_barrier(0);
            }
        aside[0] = sum + lseg, aside[1] = m;
        lseg = 0.0f, put = true;
    };
    // piece j of KS of a half's probabilities, and their images
    auto probs = [&](const f32x16_t& s, float base, int j, uint32_t (&hi)[8], uint32_t (&lo)[8]) {
#pragma unroll
        for (int u = 8 / KS * j; u < 8 / KS * (j + 1); ++u) {
            const float x = exp2_hw(s[2 * u] - base), y = exp2_hw(s[2 * u + 1] - base);
            l += x, l += y;
            split2(x, y, hi[u], lo[u]);
            asm volatile("" : "+v"(hi[u]), "+v"(lo[u]), "+v"(l));  // here, not where they are used
        }
    };
    auto part = [](const uint32_t (&x)[8], int j) { return u32x4_t{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]}; };
    // A chunk in four rows of KS steps (2 DT is as many), each of two matrix
    // instructions, a read of LDS for those two steps on, and a share of the vector
    // work: half 0's scores with the next chunk's rows to LDS; half 1's with half 0's
    // probabilities; half 0's context with half 1's; half 1's.
    static_assert(KS == 2 * DT && 8 % KS == 0);
    auto step_end = [] { __builtin_amdgcn_sched_barrier(0); };
    for (int c = r0; c < r1; c += CR, buf ^= 1) {
        u32x4_t x[3], y[3];
        x[0] = keys(0, 0), x[1] = keys(0, 1);
        uint64_t there = ~0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) there &= *(LP_LDS u64_any*)(ll + M::kFlags + buf * 32 + i * 8);
        const int next = ask_page(c + 3 * CR);
        f32x16_t s0 = zero();
        store_begin(Finite(), buf ^ 1, c + CR, pg);
        step_end();
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            x[(j + 2) % 3] = keys((j + 2) / KS, (j + 2) % KS);
            s0 = mfma32(x[j % 3], qh[j], s0);
            s0 = mfma32(x[j % 3], ql[j], s0);
            store_piece(buf ^ 1, j);
            step_end();
        }
        load_next(c + 2 * CR);
        if (c < wvis) {
            const bool whole = c + CR <= wall && __builtin_amdgcn_readfirstlane((int)(there == ~0ull));
            if (!whole) mask(c, 0, s0);
            float mx = top(s0);
            if (__ballot(mx > m + (kLift + kSlack))) scale(raise(mx));
            // (the wave that is further goes first: 12 sequences' 80 rows 40.8 us without, 39.3
            // with it, 2,048 tokens behind 14,000 852 and 832, two of 1,000 of dim 64 117 and
            // 111; without context, 2,048 tokens or six prompts, both 84 and 55.8)
            __builtin_amdgcn_s_setprio(1);
            float base = m == -INFINITY ? 0.0f : m;
            uint32_t hi[8], lo[8];
            f32x16_t s1 = zero();
            step_end();
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                if (j + 2 < KS)
                    x[(KS + j + 2) % 3] = keys(1, j + 2);
                else
                    y[j + 2 - KS] = values(j + 2 - KS);
                s1 = mfma32(x[(KS + j) % 3], qh[j], s1);
                s1 = mfma32(x[(KS + j) % 3], ql[j], s1);
                probs(s0, base, j, hi, lo);
                step_end();
            }
            if (!whole) mask(c, 1, s1);
            mx = top(s1);
            const bool up = __ballot(mx > m + (kLift + kSlack));
            float f = 1.0f;
            if (up) f = raise(mx);
            base = m == -INFINITY ? 0.0f : m;
            uint32_t hi1[8], lo1[8];
            step_end();
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                y[(i + 2) % 3] = values(i + 2);
                acc[i % DT] = mfma32(y[i % 3], part(hi, i / DT), acc[i % DT]);
                acc[i % DT] = mfma32(y[i % 3], part(lo, i / DT), acc[i % DT]);
                probs(s1, base, i, hi1, lo1);
                step_end();
            }
            if (up) scale(f);
            step_end();
#pragma unroll
            for (int i = KS; i < 2 * KS; ++i) {
                if (i + 2 < 2 * KS) y[(i + 2) % 3] = values(i + 2);
                acc[i % DT] = mfma32(y[i % 3], part(hi1, i / DT - 2), acc[i % DT]);
                acc[i % DT] = mfma32(y[i % 3], part(lo1, i / DT - 2), acc[i % DT]);
                step_end();
            }
        }
        __builtin_amdgcn_s_setprio(0);
        const int done = (c - r0) / CR + 1;  // (a chunk that some do not see says nothing)
        if ((done % kLook == 0 || done == 1 || done == 2 || done == 4) && c + CR <= wall) look(done <= kLook ? (done + 1) / 2 : kLook);
        if (!Q4 && special(c + 2 * CR, pg)) mend(Finite(), c + 2 * CR, pg);
        pg1 = page_for(next, c + 3 * CR);
        __syncthreads();
    }
    // ---- values that are no finite numbers: again, these alone, row by row and each
    // for the queries that see it (a product with 0 would make a NaN of those of others)
    if (!none) {
        if (lane == 0) *(LP_LDS u32_any*)(ll + M::kFlags + 64 + wave * 4) = 0;
        if (__ballot(strange) && lane == 0) *(LP_LDS u32_any*)(ll + M::kFlags + 64 + wave * 4) = 1;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= *(LP_LDS u32_any*)(ll + M::kFlags + 64 + i * 4);
        buf = 0;
        if (__builtin_amdgcn_readfirstlane(any))
#pragma unroll 1
            for (int c = r0; c < r1; c += CR) {
                pg = page_for(ask_page(c), c);
                load_rows(kreg, ks, a.c.k_pages, c, pg);
                load_rows(vreg, vs, a.c.v_pages, c, pg);
                if (!Q4) mend(Odd(), c, pg);
                store_rows(Odd(), 0, c, pg);
                __syncthreads();
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    if (c + 32 * t >= wvis) break;
                    f32x16_t s = zero();
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        const u32x4_t k = keys(t, j);
                        s = mfma32(k, qh[j], s);
                        s = mfma32(k, ql[j], s);
                    }
                    mask(c, t, s);
                    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = exp2_hw(s[r] - base);
#pragma unroll 1
                    for (int i = 0; i < 32; ++i) {
                        const int r = i >> 1, rr = 32 * t + 8 * (r / 4) + 4 * (i & 1) + r % 4;
                        const float pk = __shfl(s[0], n + 32 * (i & 1), 64);
                        const uint32_t at = (uint32_t)(CR * RSK + rr * RSV + 8 * h);
                        if (c + rr <= last)
#pragma unroll
                            for (int d = 0; d < DT; ++d)
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const uint32_t x = *(LP_LDS u16_any*)(ll + at + 2 * (32 * d + 8 * (e / 4) + e % 4));
                                    if (x) acc[d][e] = __builtin_fmaf(pk, f16_bits_to_f32(x), acc[d][e]);
                                }
                        if (i & 1)  // the next two rows' probabilities
#pragma unroll
                            for (int e = 0; e < 15; ++e) s[e] = s[e + 1];
                    }
                }
                __syncthreads();
            }
    }
    const Place p = place();
    if (!p.on) return;  // the halves of a query row are on or off together
    l += lseg;
    float fput = 1.0f;
    if (put) l += sum_aside(fput);
    l += shfl_xor(l, 32);
    const float f = !p.direct ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f32x4_t x = part4(d, e);
            if (put) x += get4(p, d, e) * fput;
            put4(p, d, e, x * f);
        }
    if (!p.direct && p.h == 0) gptr_w<float2>(rec_sums<D>(a))[p.rec] = make_float2(m, l);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_f16_d64(const AttnPagedArgs a) { many_body<64, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_f16_d128(const AttnPagedArgs a) { many_body<128, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_q4_d64(const AttnPagedArgs a) { many_body<64, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_q4_d128(const AttnPagedArgs a) { many_body<128, true>(a); }

// The records of a query row of a sequence with several splits, joined: a wave
// per row, its lanes the weights 2^(m_s - M), then D / 64 columns each.
namespace {

template <int D>
__device__ __forceinline__ void join_body(const AttnPagedArgs& a) {
    const int w = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = lane_id();
    const int bg = w / a.rows, row = w - bg * a.rows, b = bg / a.c.kv_heads, g = bg - b * a.c.kv_heads;
    if (b >= a.batch) return;
    const SeqView sv = seq_view(a, b);
    const int nrows = sv.n * a.group;
    if (row >= nrows) return;
    // the rows that its workgroup walked
    const int vis = seen_rows(a, sv, min(row / kManyRows * kManyRows + kManyRows, nrows) - 1);
    if (vis <= a.span) return;  // written directly
    const int S = __builtin_amdgcn_readfirstlane((vis + a.span - 1) / a.span);
    const uint64_t r0 = rec_index(a, bg, 0, row);
    float2 x = make_float2(-INFINITY, 0.0f);
    if (lane < S) x = gptr<float2>(rec_sums<D>(a))[r0 + (uint64_t)(uint32_t)lane * (uint32_t)a.rows];
    const float M = wave_max(x.x);
    const float f = x.x == -INFINITY ? 1.0f : exp2_hw(x.x - M);
    float L = f * x.y;
    for (int o = 32; o >= 1; o >>= 1) L += shfl_xor(L, o);
    constexpr int C = D / 64;
    float A[C] = {};
    // sixteen records' loads at a time, for they are what this takes (512 rows of 59
    // records 8.4 us, eight at a time 17)
    for (int s0 = 0; s0 < S; s0 += 16) {
        float x[16][C];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            if (s0 + u >= S) break;
            const uint64_t at = a.part + (r0 + (uint64_t)(uint32_t)(s0 + u) * (uint32_t)a.rows) * (D * 4);
            if constexpr (C == 2) {
                const float2 v = gptr<float2>(at)[lane];
                x[u][0] = v.x, x[u][1] = v.y;
            } else {
                x[u][0] = gptr<float>(at)[lane];
            }
        }
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (s0 + u < S) {
                const float fs = __shfl(f, s0 + u, 64);
#pragma unroll
                for (int i = 0; i < C; ++i) A[i] = __builtin_fmaf(fs, x[u][i], A[i]);
            }
    }
    const int i = row / a.group, h = g * a.group + (row - i * a.group);
    const uint64_t o = a.out + ((uint64_t)(uint32_t)(sv.t0 + i) * (uint32_t)a.out_stride + (uint32_t)(h * D)) * 4;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if constexpr (C == 2)
        gptr_w<float2>(o)[lane] = make_float2(A[0] * inv, A[1] * inv);
    else
        gptr_w<float>(o)[lane] = A[0] * inv;
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_attn_join_d64(const AttnPagedArgs a) { join_body<64>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_join_d128(const AttnPagedArgs a) { join_body<128>(a); }
