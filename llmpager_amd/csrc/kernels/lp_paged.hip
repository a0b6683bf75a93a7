// gfx950 kernels of a batch's KV cache in pages: the append of new tokens and their
// causal attention (lp_paged_device.h has the bodies, and why they are as they are).
#include "lp_paged_device.h"

extern "C" __global__ void __launch_bounds__(256) lp_kv_append_f16_d64(const KvAppendPagedArgs a) { append_body<64, false, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_f16_d128(const KvAppendPagedArgs a) { append_body<128, false, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_q4_d64(const KvAppendPagedArgs a) { append_body<64, true, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_kv_append_q4_d128(const KvAppendPagedArgs a) { append_body<128, true, false>(a); }

// (waves a SIMD that the registers leave room for; with 4-bit rows of 128 the second set
// of sums takes the third: 256 sequences' 4 KV heads over up to 2,000 rows 67 us, 62 with
// three and one set, 95 with three and both, spilled)
#define LP_ATTN_FEW(NAME, WAVES, D, Q4, NT) \
    extern "C" __global__ void __launch_bounds__(256, WAVES) lp_attn_few_##NAME(const AttnPagedArgs a) { few_body<D, Q4, NT, false>(a); }
LP_ATTN_FEW(f16_d64, 2, 64, false, 1)
LP_ATTN_FEW(f16_d128, 2, 128, false, 1)
LP_ATTN_FEW(q4_d64, 3, 64, true, 1)
LP_ATTN_FEW(q4_d128, 2, 128, true, 1)
LP_ATTN_FEW(f16_d64_n2, 2, 64, false, 2)
LP_ATTN_FEW(f16_d128_n2, 1, 128, false, 2)
LP_ATTN_FEW(q4_d64_n2, 2, 64, true, 2)
LP_ATTN_FEW(q4_d128_n2, 1, 128, true, 2)
#undef LP_ATTN_FEW

extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_f16_d64(const AttnPagedArgs a) { many_body<64, false, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_f16_d128(const AttnPagedArgs a) { many_body<128, false, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_q4_d64(const AttnPagedArgs a) { many_body<64, true, false>(a); }
extern "C" __global__ void __launch_bounds__(256, 2) lp_attn_many_q4_d128(const AttnPagedArgs a) { many_body<128, true, false>(a); }

extern "C" __global__ void __launch_bounds__(256) lp_attn_join_d64(const AttnPagedArgs a) { join_body<64, false>(a); }
extern "C" __global__ void __launch_bounds__(256) lp_attn_join_d128(const AttnPagedArgs a) { join_body<128, false>(a); }
