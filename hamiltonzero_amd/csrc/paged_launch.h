// Host-side launch interface of the paged operators (include/hz_paged.h) between the C ABI
// (mhsea_abi.hip) and the kernel files, and what the kernels share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/hz_paged.h"

namespace hz {

// qk_norm_rotary.hip.
int64_t qk_rotary_workspace(int64_t tokens, int64_t D, bool norm);
hipError_t launch_qk_rotary_fwd(const hz_qk_rotary& p, hipStream_t stream);
hipError_t launch_qk_rotary_bwd(const hz_qk_rotary& p, void* dq, void* dk, float* dw_q, float* dw_k, void* workspace,
                                hipStream_t stream);

// paged_attention.hip.
int64_t paged_attention_workspace(const hz_paged_attention_args& p);
hipError_t launch_paged_attention(const hz_paged_attention_args& p, void* workspace, hipStream_t stream);

// paged_cache.hip.
hipError_t launch_paged_append(const hz_paged_cache& c, const hz_token_tensor& k, const hz_token_tensor& v, int64_t N,
                               hipStream_t stream);
int64_t paged_evict_workspace(const hz_paged_evict_args& p);
hipError_t launch_paged_evict(const hz_paged_evict_args& p, void* workspace, hipStream_t stream);

// A cache's rows of slots as the kernels read them.
struct Pages {
  const int32_t *table, *lengths;
  int64_t page_k, token_k, head_k, page_v, token_v, head_v;  // strides in elements
  const void *k, *v;
  int pages, size, width, slots;  // slots of a row: width * size
  uint32_t by_size;               // ceil(2^32 / size), for size > 1
  explicit Pages(const hz_paged_cache& c)
      : table(c.page_table), lengths(c.lengths), page_k(c.k.batch), token_k(c.k.token), head_k(c.k.head),
        page_v(c.v.batch), token_v(c.v.token), head_v(c.v.head), k(c.k.data), v(c.v.data),
        pages(static_cast<int>(c.pages)), size(static_cast<int>(c.page_size)), width(static_cast<int>(c.table_width)),
        slots(pages_slots(c)), by_size(c.page_size > 1 ? static_cast<uint32_t>(((int64_t(1) << 32) + c.page_size - 1) / c.page_size) : 0) {}
  static int pages_slots(const hz_paged_cache& c) { return static_cast<int>(c.page_size * c.table_width); }

  __device__ __forceinline__ int length(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : n > slots ? slots : n;
  }
  // slot / size. The quotient by the rounded-up reciprocal is the right one or one too large: slot < 2^30.
  __device__ __forceinline__ int page_of(int slot) const {
    if (by_size == 0) return slot;
    const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(slot), by_size));
    return q * size > slot ? q - 1 : q;
  }
};

// x of this lane and all before it. (Unsigned: two numbers of sixteen bits are summed as one.)
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  auto from = [&](auto control, auto rows) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), control.value, rows.value, 0xf, false));
  };
  typedef std::integral_constant<int, 0xf> All;
  x += from(std::integral_constant<int, 0x111>{}, All{});  // from 1, 2, 4 and 8 lanes below in the row of sixteen
  x += from(std::integral_constant<int, 0x112>{}, All{});
  x += from(std::integral_constant<int, 0x114>{}, All{});
  x += from(std::integral_constant<int, 0x118>{}, All{});
  x += from(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // the row's last lane to the next row, of rows 1 and 3
  x += from(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // lane 31 to rows 2 and 3
  return x;
}

}  // namespace hz
