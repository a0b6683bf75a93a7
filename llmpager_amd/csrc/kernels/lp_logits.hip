// gfx950 kernels that read rows of logits: log probabilities of given tokens,
// the rows' entropies and their top alternatives.
//
// With M the row's largest logit, S = sum e^(x - M) and Y = sum e^(x - M) (x - M):
//   log p(x) = (x - M) - log S,   entropy = log S - Y / S.
// S and Y are summed in 64 bits: in a row that is sure of one token the entropy
// is all in what the other terms add to the 1 of the largest.
#include "lp_device.h"

using namespace lp;
using namespace lpk;

namespace {

__device__ __forceinline__ double wave_sum_f64(double v) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

}  // namespace

// A workgroup per row: its largest value, its sums, then one pass per
// alternative for the next in the order (value, lowest index first).
extern "C" __global__ void __launch_bounds__(256) lp_logprobs(const LogprobArgs a) {
    __shared__ float redf[4];
    __shared__ int redi[4];
    __shared__ double redd[2][4];
    const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
    const LP_GLOBAL float* x = gptr<float>(a.logits + (uint64_t)row * (uint32_t)a.stride * 4);
    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += 256) m = fmaxf(m, x[i]);
    m = wave_max(m);
    if (lane_id() == 0) redf[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3]));
    double s = 0.0, y = 0.0;
    for (int i = tid; i < a.vocab; i += 256) {
        const float d = x[i] - m;
        const float e = expf(d);
        s += (double)e;
        y += d == -INFINITY ? 0.0 : (double)e * (double)d;
    }
    s = wave_sum_f64(s);
    y = wave_sum_f64(y);
    if (lane_id() == 0) redd[0][wave] = s, redd[1][wave] = y;
    __syncthreads();
    s = redd[0][0] + redd[0][1] + redd[0][2] + redd[0][3];
    y = redd[1][0] + redd[1][1] + redd[1][2] + redd[1][3];
    const double lse = log(s);
    if (tid == 0) {
        if (a.targets) {
            const int t = gptr<int>(a.targets)[row];
            gptr_w<float>(a.logp)[row] = (uint32_t)t < (uint32_t)a.vocab ? (float)((double)(x[t] - m) - lse) : 0.0f;
        }
        if (a.entropy) gptr_w<float>(a.entropy)[row] = (float)(lse - y / s);
    }
    float pv = INFINITY;
    int pi = -1;
    for (int k = 0; k < a.top; ++k) {
        float bv = -INFINITY;
        int bi = INT32_MAX;
        for (int i = tid; i < a.vocab; i += 256) {
            const float v = x[i];
            const bool next = v < pv || (v == pv && i > pi);
            if (next && (v > bv || (v == bv && i < bi))) bv = v, bi = i;
        }
        for (int o = 32; o >= 1; o >>= 1) {
            const float ov = shfl_xor(bv, o);
            const int oi = __shfl_xor(bi, o, 64);
            if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
        }
        __syncthreads();
        if (lane_id() == 0) redf[wave] = bv, redi[wave] = bi;
        __syncthreads();
        for (int w = 0; w < 4; ++w)
            if (redf[w] > bv || (redf[w] == bv && redi[w] < bi)) bv = redf[w], bi = redi[w];
        pv = bv, pi = bi;
        if (tid == 0) {
            const bool none = bi == INT32_MAX;
            gptr_w<int>(a.ids)[(uint64_t)row * (uint32_t)a.top + k] = none ? -1 : bi;
            gptr_w<float>(a.top_logp)[(uint64_t)row * (uint32_t)a.top + k] =
                none ? __builtin_nanf("") : (float)((double)(bv - m) - lse);
        }
    }
}
