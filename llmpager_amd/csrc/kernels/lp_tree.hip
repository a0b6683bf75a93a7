// gfx950 kernels of a step whose new tokens are trees of drafts: depths and ancestors of
// their nodes (lp_tree_layout), the append and the attention of lp_paged_device.h
// where depths and masks take the place of positions (lp_kv_append_tree_*,
// lp_attn_tree_*), and the rows of the tokens that stay moved together (lp_kv_keep_*).
#include "lp_paged_device.h"

// Append: the angles are the depths', the rest that of lp_paged.hip and bound like it, by the
// launch or the copy rate: 1,273 tokens of 32 sequences, 64 + 2 x 4 heads of 128, 16-bit
// pages: 22 us, 4.2 TB/s of 91 MB (17.3 us at the rate of a large copy).
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_tree_f16_d64(const KvAppendPagedArgs a) { append_body<64, false, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_tree_f16_d128(const KvAppendPagedArgs a) { append_body<128, false, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_tree_q4_d64(const KvAppendPagedArgs a) { append_body<64, true, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_tree_q4_d128(const KvAppendPagedArgs a) { append_body<128, true, true>(a); }

// Attention: a chunk of rows before the new ones is walked as in lp_paged.hip, one that
// holds new ones has each query row's scores taken from its token's mask.  26 tokens of 32
// heads on 4 of 128 over 1,526 16-bit rows 16.6 us: the launch, a chain of round trips
// (lengths, pages, rows), three units a workgroup and the join of up to 4 parts.  16 sequences of up to 32 tokens,
// up to 6,032 4-bit rows: 70 us and 10 of the join; its 8,212 chunks of 128 query rows by 64 are 59 us of matrix
// work on 256 CUs, of which the fullest has 36 and the mean 32.  27 % of the chunks' query rows are none (96 to
// 256 rows a sequence and KV head), 20 % of their waves have none at all, which do a quarter of
// a full one's matrix work still: by the waves that have some it would be 47 us.  4 sequences of up to 256 tokens, 64 heads on
// 4, 3,257 16-bit rows and fewer: 135 us, 15,612 chunks, 112 us of matrix work, 73 chunks on the fullest CU and
// 61 on the mean; parts of them cost more in records and joins than they even out (1,024 workgroups
// 164 us where 512 took 163, of the 16 sequences 93 against 87).
// (waves a SIMD as in lp_paged.hip)
#define LP_ATTN_TREE_FEW(NAME, WAVES, D, Q4, NT) \
    extern "C" __global__ void __launch_bounds__(256, WAVES) lp_attn_tree_few_##NAME(const AttnPagedArgs a) { few_body<D, Q4, NT, true>(a); }
LP_ATTN_TREE_FEW(f16_d64, 2, 64, false, 1)
LP_ATTN_TREE_FEW(f16_d128, 2, 128, false, 1)
LP_ATTN_TREE_FEW(q4_d64, 3, 64, true, 1)
LP_ATTN_TREE_FEW(q4_d128, 2, 128, true, 1)
LP_ATTN_TREE_FEW(f16_d64_n2, 2, 64, false, 2)
LP_ATTN_TREE_FEW(f16_d128_n2, 1, 128, false, 2)
LP_ATTN_TREE_FEW(q4_d64_n2, 2, 64, true, 2)
LP_ATTN_TREE_FEW(q4_d128_n2, 1, 128, true, 2)
#undef LP_ATTN_TREE_FEW

extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_tree_many_f16_d64(const AttnPagedArgs a) { many_body<64, false, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_tree_many_f16_d128(const AttnPagedArgs a) { many_body<128, false, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_tree_many_q4_d64(const AttnPagedArgs a) { many_body<64, true, true>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_tree_many_q4_d128(const AttnPagedArgs a) { many_body<128, true, true>(a); }

extern "C" __global__ void __launch_bounds__(256) lp_attn_tree_join_d64(const AttnPagedArgs a) { join_body<64, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_tree_join_d128(const AttnPagedArgs a) { join_body<128, true>(a); }

// ---------------------------------------------------------------------------
// Layout.  A workgroup takes one 64-bit word of a sequence's masks.  A node points
// to its parent and holds its own bit and the distance 1; each round every node takes
// over what the node that it points to has gathered and points where that does, twice as far
// up, so a tree of depth d is done after log2 d + 1 rounds.  A launch's time: 64 trees of up to 60
// nodes 5.0 us from the host, where an empty kernel takes 4 to 5.
// ---------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256) lp_tree_layout(const TreeLayoutArgs a) {
    __shared__ uint64_t mask[kTreeMaxNodes];
    __shared__ int up[kTreeMaxNodes], depth[kTreeMaxNodes];
    constexpr int N = kTreeMaxNodes / 256;
    const int b = (int)blockIdx.x / a.words, w = (int)blockIdx.x - b * a.words;
    const int t0 = gptr<int>(a.q_starts)[b], n = min(gptr<int>(a.q_starts)[b + 1] - t0, a.max_q);
    if (n <= 0 || t0 < 0 || t0 > a.tokens - n) return;  // starts that name no tokens
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = (int)threadIdx.x + 256 * k;
        if (i >= n) continue;
        const int p = gptr<int>(a.parents)[t0 + i];
        const bool has = p >= 0 && p < i;
        up[i] = has ? p : -1;
        depth[i] = has;
        mask[i] = i >> 6 == w ? 1ull << (i & 63) : 0;
    }
    __syncthreads();
    for (int round = 0; round < 32 - __builtin_clz(kTreeMaxNodes); ++round) {
        int u[N], d[N];
        uint64_t m[N];
        bool on = false;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = (int)threadIdx.x + 256 * k;
            u[k] = i < n ? up[i] : -1;
            if (u[k] < 0) continue;
            on = true;
            d[k] = depth[u[k]], m[k] = mask[u[k]], u[k] = up[u[k]];
            d[k] += depth[i], m[k] |= mask[i];
            if (u[k] < 0) u[k] = -2;  // done, to be written still
        }
        if (!__syncthreads_or(on)) break;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = (int)threadIdx.x + 256 * k;
            if (i < n && u[k] != -1) depth[i] = d[k], mask[i] = m[k], up[i] = max(u[k], -1);
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = (int)threadIdx.x + 256 * k;
        if (i >= n) continue;
        gptr_w<uint64_t>(a.masks)[(uint64_t)(uint32_t)(t0 + i) * (uint32_t)a.words + (uint32_t)w] = mask[i];
        if (w == 0) gptr_w<int>(a.depths)[t0 + i] = depth[i];
    }
}

// ---------------------------------------------------------------------------
// Keep.  Row p0 + i of a sequence takes row p0 + path[i], in both pools of a layer, for
// every KV head.  A wave has a share of a row's units (16 bytes, 4 of 4-bit rows) and moves
// them for all of the path, four rows read before they are written: path rises, so a row
// that is written is none that is still to be read.  All layers are one launch, its arguments
// hold their pools: 64 sequences, up to 9 rows of 4 heads of 128 in 48 layers, 16 bits: 5.3 us, a launch's
// time (a launch a layer would be 48 of these).
// ---------------------------------------------------------------------------
namespace {

template <int D, bool Q4>
__device__ __forceinline__ void keep_body(const KvKeepArgs& a) {
    constexpr int UB = Q4 ? 4 : 16, SU = Q4 ? D / 64 : 0, U = SU + (Q4 ? D / 2 : D * 2) / UB;  // bytes of a unit; of scales; of a row
    constexpr int K = keep_units(Q4) / 64, R = 4;
    using Unit = std::conditional_t<Q4, uint32_t, u32x4_t>;
    const int lane = lane_id(), w = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
    const int chunk = w % a.chunks, b = w / a.chunks / a.layers, layer = w / a.chunks - b * a.layers;
    if (b >= a.batch) return;
    const int n = gptr<int>(a.q_starts)[b + 1] - gptr<int>(a.q_starts)[b];
    const int p0 = gptr<int>(a.seq_lens)[b] - n, k = max(0, min(gptr<int>(a.kept)[b], min(n, a.max_depth + 1)));
    if (a.lens_out && layer == 0 && chunk == 0 && lane == 0) gptr_w<int>(a.lens_out)[b] = p0 + k;
    uint64_t at[K];  // a unit's place in row 0 of page 0, and what a row adds to it
    uint32_t step[K];
    bool on[K];
    const uint64_t kp = a.k_pages[layer], vp = a.v_pages[layer];
    const uint32_t pbytes = (uint32_t)page_bytes(D, 1 << a.c.page_log2, Q4);
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int u = chunk * (64 * K) + 64 * i + lane, head = u / U, piece = u - head * U, g = head >> 1;
        on[i] = g < a.c.kv_heads;
        step[i] = piece < SU ? SU * 4 : Q4 ? D / 2 : D * 2;
        at[i] = pick(head & 1, vp, kp) + (uint64_t)(uint32_t)g * pbytes +
                (piece < SU ? 4 * piece : ((uint32_t)(SU * 4) << a.c.page_log2) + UB * (piece - SU));
    }
    const uint64_t page_step = (uint64_t)pbytes * (uint32_t)a.c.kv_heads;
    const int pmask = (1 << a.c.page_log2) - 1;
    for (int i0 = 0; i0 < k; i0 += 64) {
        const int i = i0 + lane;
        int x = -1, from = -1, to = -1;
        if (i < k) x = gptr<int>(a.path)[(uint64_t)(uint32_t)b * (uint32_t)(a.max_depth + 1) + (uint32_t)i];
        if (x >= 0 && x < n && x != i) from = page_of(a.c, b, p0 + x), to = page_of(a.c, b, p0 + i);
        for (uint64_t move = __ballot(from >= 0 && to >= 0); move;) {
            Unit v[R][K];
            const uint64_t these = move;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (!move) continue;
                const int l = __builtin_ctzll(move), row = p0 + __builtin_amdgcn_readlane(x, l);
                const uint64_t src = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(from, l) * page_step;
                move &= move - 1;
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (on[j]) v[r][j] = *gptr<Unit>(at[j] + src + (uint32_t)(row & pmask) * step[j]);
            }
            move = these;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (!move) continue;
                const int l = __builtin_ctzll(move), row = p0 + i0 + l;
                const uint64_t dst = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(to, l) * page_step;
                move &= move - 1;
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (on[j]) *gptr_w<Unit>(at[j] + dst + (uint32_t)(row & pmask) * step[j]) = v[r][j];
            }
        }
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) lp_kv_keep_f16_d64(const KvKeepArgs a) { keep_body<64, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_keep_f16_d128(const KvKeepArgs a) { keep_body<128, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_keep_q4_d64(const KvKeepArgs a) { keep_body<64, true>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_keep_q4_d128(const KvKeepArgs a) { keep_body<128, true>(a); }
