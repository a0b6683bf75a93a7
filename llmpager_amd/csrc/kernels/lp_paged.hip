// gfx950 kernels of a batch's KV cache in pages: the new tokens' queries and
// keys normed per head and rotated with keys and values written into their
// pages (lp_kv_append_*), and attention of one or many new tokens a sequence
// over its pages (lp_attn_paged_*).
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

// The token's sequence (batch for a token behind the last one): the sequences
// that end at or before it.
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
// whatever the order of the sums.
// ---------------------------------------------------------------------------
template <int D, bool Q4>
__device__ __forceinline__ void append_body(const KvAppendPagedArgs& a) {
    constexpr int LPR = D / 4, RPW = 64 / LPR, G = D / 32;
    const int lane = lane_id(), j = lane % LPR, sub = lane / LPR;
    const int w = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    const int token = w / a.parts;
    if (token >= a.tokens) return;  // whole waves
    const int b = sequence_of(a.q_starts, a.batch, token);
    if (b >= a.batch) return;  // behind the last sequence: left as it was
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
        sincos(r, &sn[u], &cs[u]);
        cs[u] *= (double)a.mscale;
        sn[u] *= (double)a.mscale;
    }
    const int H = a.heads, KV = a.c.kv_heads, rows = H + 2 * KV;
    const int r1 = min(rows, (w % a.parts + 1) * a.rows_per_part);
    for (int r = w % a.parts * a.rows_per_part; r < r1; r += RPW) {
        const int row = r + sub;
        const bool on = row < r1, isq = row < H, isk = !isq && row < H + KV;
        const int head = isq ? row : isk ? row - H : row - H - KV;
        const uint64_t src = (isq ? a.q : isk ? a.k : a.v) +
                             ((uint64_t)token * (uint32_t)(isq ? a.q_stride : isk ? a.k_stride : a.v_stride) +
                              (uint32_t)(head * D)) * 4;
        float2 f0 = make_float2(0.0f, 0.0f), f1 = f0, w0 = make_float2(1.0f, 1.0f), w1 = w0;
        if (on) {
            f0 = gptr<float2>(src)[j];
            f1 = gptr<float2>(src)[LPR + j];
            const uint64_t nw = isq ? a.q_norm : isk ? a.k_norm : 0;
            if (nw) {
                w0 = gptr<float2>(nw)[j];
                w1 = gptr<float2>(nw)[LPR + j];
            }
        }
        double x[4] = {f0.x, f0.y, f1.x, f1.y};
        double ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
        ss = row16_f64(ss, [](double p, double q) { return p + q; });
        if constexpr (LPR == 32) ss += __shfl_xor(ss, 16, 64);
        if (isq || isk) {
            if (isq ? a.q_norm != 0 : a.k_norm != 0) {
                const double inv = 1.0 / sqrt(ss / (double)D + (double)a.eps);
                x[0] *= inv * (double)w0.x;
                x[1] *= inv * (double)w0.y;
                x[2] *= inv * (double)w1.x;
                x[3] *= inv * (double)w1.y;
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
        float2 held[2];
        const uint64_t pg = page_at<D, Q4>(a.c, isk ? a.c.k_pages : a.c.v_pages, max(page, 0), isq ? 0 : head);
        const bool store = on && !isq && page >= 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const double x0 = x[2 * u], x1 = x[2 * u + 1];
            if constexpr (Q4) {
                // the group's scale; a NaN counts as zero, so that a 4-bit row holds numbers only
                const double m = row16_f64(fmax(fmax(fabs(x0), fabs(x1)), 0.0), [](double p, double q) { return fmax(p, q); });
                const double s = fmin(fmax(round7(m / 7.0), kQ4MinScale), kQ4MaxScale);
                const int c0 = x0 == x0 ? (int)fmin(fmax(rint(x0 / s), -7.0), 7.0) : 0;
                const int c1 = x1 == x1 ? (int)fmin(fmax(rint(x1 / s), -7.0), 7.0) : 0;
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
        const uint64_t ko = isk ? a.k_out : a.v_out;
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

// ---------------------------------------------------------------------------
// Attention, a wave per (query token, head): 64 rows at a time, a row's score
// per lane, an online softmax over the rows, then the context with the
// dimensions across the lanes.
// ---------------------------------------------------------------------------
namespace {

template <int D, bool Q4>
__device__ __forceinline__ float row_value(uint64_t page, int log2, int row, int d) {
    if constexpr (Q4) {
        const float s = f16_bits_to_f32(gptr<uint16_t>(page)[row * (D / 32) + d / 32]);
        const uint32_t n = gptr<uint8_t>(page + (uint32_t)(D / 16 << log2))[row * (D / 2) + d / 2];
        return s * (float)((int)(n >> (4 * (d & 1)) & 15) - 8);
    } else {
        return f16_bits_to_f32(gptr<uint16_t>(page)[row * D + d]);
    }
}

template <int D, bool Q4>
__device__ __forceinline__ void attn_body(const AttnPagedArgs& a) {
    __shared__ float qs[4][D];
    const int wave = (int)(threadIdx.x >> 6), lane = lane_id();
    const int w = (int)blockIdx.x * 4 + wave;
    const int h = w % a.heads, i = w / a.heads % a.max_q, b = w / a.heads / a.max_q;
    if (b >= a.batch) return;
    const int t0 = gptr<int>(a.q_starts)[b], n = gptr<int>(a.q_starts)[b + 1] - t0, t = t0 + i;
    if (i >= n || t < 0 || t >= a.tokens) return;
    const int len = min(gptr<int>(a.seq_lens)[b], a.max_seq);
    const int pos = len - n + i, g = h / a.group;
    const uint64_t q = a.q + ((uint64_t)t * (uint32_t)a.q_stride + (uint32_t)(h * D)) * 4;
    for (int d = lane; d < D; d += 64) qs[wave][d] = gptr<float>(q)[d];
    __builtin_amdgcn_wave_barrier();
    constexpr int DL = D / 64;
    float m = -INFINITY, l = 0.0f, acc[DL] = {};
    for (int r0 = 0; r0 <= pos; r0 += 64) {
        const int row = r0 + lane;
        const int pg = row <= pos ? page_of(a.c, b, row) : -1;
        const int pr = row & ((1 << a.c.page_log2) - 1);
        float s = -INFINITY;
        if (pg >= 0) {
            const uint64_t at = page_at<D, Q4>(a.c, a.c.k_pages, pg, g);
            s = 0.0f;
            for (int d = 0; d < D; ++d) s = __builtin_fmaf(qs[wave][d], row_value<D, Q4>(at, a.c.page_log2, pr, d), s);
            s *= a.scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float alpha = mn == -INFINITY ? 1.0f : expf(m - mn);
        const float p = pg < 0 || mn == -INFINITY ? 0.0f : expf(s - mn);
        float sum = p;
        for (int o = 32; o >= 1; o >>= 1) sum += shfl_xor(sum, o);
        l = __builtin_fmaf(l, alpha, sum);
        m = mn;
#pragma unroll
        for (int u = 0; u < DL; ++u) acc[u] *= alpha;
        uint64_t seen = __ballot(pg >= 0);
        while (seen) {
            const int k = __builtin_ctzll(seen);
            seen &= seen - 1;
            const float pk = __shfl(p, k, 64);
            const uint64_t at = page_at<D, Q4>(a.c, a.c.v_pages, __shfl(pg, k, 64), g);
            const int kr = (r0 + k) & ((1 << a.c.page_log2) - 1);
#pragma unroll
            for (int u = 0; u < DL; ++u)
                acc[u] = __builtin_fmaf(pk, row_value<D, Q4>(at, a.c.page_log2, kr, lane + 64 * u), acc[u]);
        }
    }
    const uint64_t o = a.out + ((uint64_t)t * (uint32_t)a.out_stride + (uint32_t)(h * D)) * 4;
#pragma unroll
    for (int u = 0; u < DL; ++u) gptr_w<float>(o)[lane + 64 * u] = l == 0.0f ? 0.0f : acc[u] / l;
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_attn_paged_f16_d64(const AttnPagedArgs a) { attn_body<64, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_paged_f16_d128(const AttnPagedArgs a) { attn_body<128, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_paged_q4_d64(const AttnPagedArgs a) { attn_body<64, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_paged_q4_d128(const AttnPagedArgs a) { attn_body<128, true>(a); }
