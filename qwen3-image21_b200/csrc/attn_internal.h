// attn_internal.h — launches of attn_fwd.cu that other files of the library build on.
// Arguments are validated by the callers.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/b200_attn.h"

namespace b200 {

// Attention of post-RoPE q [B,H,T,128] over [prefix (B,H,P,128) ; k_rot (B,H,T,128) and
// v (B,T,H,128)], out [B,T,H*128].  split_region: B200_ATTN_SPLIT_WORKSPACE_BYTES of
// scratch for the tail split, or NULL.
int joint_attention(const void* q_rot, const void* k_rot, const void* v, const void* prefix_k,
                    const void* prefix_v, int B, int H, int T, int P, const b200_kv_desc* desc,
                    float scale, void* out, int32_t* status, void* split_region,
                    cudaStream_t stream, bool counters_zeroed = false,
                    const int32_t* row_limit = nullptr);

// The arrival counters of a split region, which are zero before the launch: `n` words that
// the caller clears where it says counters_zeroed.
int32_t* split_counters(void* split_region, int* n);

// Q/K RMSNorm + RoPE of args (and the copy of V to v_out, if given) into q_rot and k_rot.
int attn_prologue(const b200_attn_args& args, void* q_rot, void* k_rot, cudaStream_t stream);

}  // namespace b200
