// Host-side launch interface of the token operators (include/hz_token.h) between the C ABI
// (mhsea_abi.hip) and the kernel files.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hz_token.h"

namespace hz {

// qk_norm_rotary.hip. The workspace holds one row of partial weight gradients a workgroup.
int64_t qk_norm_rotary_workspace(int64_t tokens, int64_t D);
hipError_t launch_qk_norm_rotary_fwd(const hz_qk_norm_rotary& p, hipStream_t stream);
hipError_t launch_qk_norm_rotary_bwd(const hz_qk_norm_rotary& p, void* dq, void* dk, float* dw_q, float* dw_k,
                                     void* workspace, hipStream_t stream);

// token_attention_fwd.hip, token_attention_bwd.hip.
int64_t token_attention_fwd_workspace(const hz_token_attention& p);
hipError_t launch_token_attention_fwd(const hz_token_attention& p, void* workspace, hipStream_t stream);
int64_t token_attention_bwd_workspace(const hz_token_attention& p);
hipError_t launch_token_attention_bwd(const hz_token_attention& p, const hz_token_tensor& dout, void* dq, void* dk,
                                      void* dv, void* workspace, hipStream_t stream);

// bucket_bias.hip.
struct BucketParams {
  const int32_t *buckets, *qpos, *kpos;
  int64_t B, Nq, Nk;
  int H, nb, R;
  bool qkh;  // e is [B, Nq, Nk, H], else [B, Nq, H, Nk]
  int dtype;
};
hipError_t launch_bucket_bias_fwd(const BucketParams& p, const float* table, void* e, hipStream_t stream);
int64_t bucket_bias_workspace(const BucketParams& p);
hipError_t launch_bucket_bias_bwd(const BucketParams& p, const void* de, float* dtable, void* workspace,
                                  hipStream_t stream);

}  // namespace hz
