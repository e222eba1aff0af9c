// Learned relative position bias by buckets, written into the attention's bias layouts, and its
// table's gradient (formulas: include/hz_token.h).
//
// Forward: one lookup in LDS an element; bound by the bytes it writes. The table is held head by
// head (a row of buckets for each head), so lanes on different buckets read different banks.
// Backward: a histogram of de by bucket, bound by the bytes it reads. Every thread adds its
// elements to a column of its own in LDS (ds_add_f32, bank = lane: no conflicts and one order of
// additions), a workgroup sums its columns at the end and a second kernel the workgroups' rows: no
// result depends on the order in which workgroups run.
#include "mhsea_device.h"
#include "token_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int bucket_of(const BucketParams& p, const uint16_t* buckets, int qpos, int kpos) {
  int64_t d = static_cast<int64_t>(kpos) - qpos;
  d = d < -p.R ? -p.R : d > p.R ? p.R : d;
  return buckets[p.R + static_cast<int>(d)];
}

// buckets to LDS; a number outside the table becomes nb, a bucket whose bias is zero.
__device__ __forceinline__ void stage_buckets(const BucketParams& p, uint16_t* buckets, int threads) {
  for (int i = threadIdx.x; i < 2 * p.R + 1; i += threads) {
    const int m = p.buckets[i];
    buckets[i] = static_cast<uint16_t>(m < 0 || m >= p.nb ? p.nb : m);
  }
}

// A thread takes the same element of every head: [B, Nq, H, Nk] (lanes along the keys).
template <class S>
__global__ void __launch_bounds__(kThreads) bucket_bias_qhk_kernel(BucketParams p, const float* table, void* e) {
  extern __shared__ float lds[];
  const int ld = p.nb + 1;
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + p.H * ld);
  for (int i = threadIdx.x; i < p.H * ld; i += kThreads) {
    const int h = i / ld, m = i - h * ld;
    lds[i] = m < p.nb ? table[static_cast<int64_t>(m) * p.H + h] : 0.f;
  }
  stage_buckets(p, buckets, kThreads);
  __syncthreads();
  const int64_t items = p.B * p.Nq * p.Nk;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; it < items;
       it += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = it / p.Nk, j = it - row * p.Nk, b = row / p.Nq;
    const int m = bucket_of(p, buckets, p.qpos[row], p.kpos[b * p.Nk + j]);
    for (int h = 0; h < p.H; ++h) store1<S>(e, (row * p.H + h) * p.Nk + j, lds[h * ld + m]);
  }
}

// [B, Nq, Nk, H]: lanes along the heads of consecutive keys.
template <class S>
__global__ void __launch_bounds__(kThreads) bucket_bias_qkh_kernel(BucketParams p, const float* table, void* e) {
  extern __shared__ float lds[];
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + (p.nb + 1) * p.H);
  for (int i = threadIdx.x; i < (p.nb + 1) * p.H; i += kThreads) lds[i] = i < p.nb * p.H ? table[i] : 0.f;
  stage_buckets(p, buckets, kThreads);
  __syncthreads();
  const int64_t items = p.B * p.Nq * p.Nk * p.H;
  for (int64_t it = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; it < items;
       it += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t pair = it / p.H, row = pair / p.Nk, j = pair - row * p.Nk, b = row / p.Nq;
    const int m = bucket_of(p, buckets, p.qpos[row], p.kpos[b * p.Nk + j]);
    store1<S>(e, it, lds[m * p.H + static_cast<int>(it - pair * p.H)]);
  }
}

// Partial gradients: partial [slots][nb][H]. qhk: grid (slots, H), every thread on head blockIdx.y; qkh: grid
// (slots), thread t on head t % H (threads behind the last whole set of heads idle).
template <class S, bool QKH>
__global__ void bucket_bias_bwd_kernel(BucketParams p, const void* de, float* partial) {
  extern __shared__ float lds[];
  const int T = blockDim.x, tid = threadIdx.x;
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + (p.nb + 1) * T);
  for (int i = tid; i < (p.nb + 1) * T; i += T) lds[i] = 0.f;
  stage_buckets(p, buckets, T);
  __syncthreads();
  float* const mine = lds + tid;
  const int h = QKH ? tid % p.H : static_cast<int>(blockIdx.y);
  const int heads = QKH ? p.H : 1;
  const int pairs = T / heads;  // pairs of query and key that a workgroup takes at a time
  const int64_t items = p.B * p.Nq * p.Nk;
  if (tid < pairs * heads)
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * pairs + tid / heads; it < items;
         it += static_cast<int64_t>(gridDim.x) * pairs) {
      const int64_t row = it / p.Nk, j = it - row * p.Nk, b = row / p.Nq;
      const int m = bucket_of(p, buckets, p.qpos[row], p.kpos[b * p.Nk + j]);
      const float x = load1<S>(de, QKH ? it * p.H + h : (row * p.H + h) * p.Nk + j);
      __hip_atomic_fetch_add(mine + m * T, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  __syncthreads();
  for (int i = tid; i < p.nb * heads; i += T) {
    const int m = i / heads, hh = i - m * heads;
    float sum = 0.f;
    for (int t = hh; t < pairs * heads; t += heads) sum += lds[m * T + t];
    partial[(static_cast<int64_t>(blockIdx.x) * p.nb + m) * p.H + (QKH ? hh : h)] = sum;
  }
}

__global__ void __launch_bounds__(kThreads) bucket_sum_kernel(const float* partial, int slots, int n, float* dtable) {
  __shared__ float red[kThreads];
  const int c = threadIdx.x % 16, r0 = threadIdx.x / 16, col = blockIdx.x * 16 + c;
  float sum = 0.f;
  if (col < n)
    for (int s = r0; s < slots; s += kThreads / 16) sum += partial[static_cast<int64_t>(s) * n + col];
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int m = kThreads / 32; m > 0; m >>= 1) {
    if (r0 < m) red[threadIdx.x] += red[threadIdx.x + m * 16];
    __syncthreads();
  }
  if (r0 == 0 && col < n) dtable[col] = red[c];
}

size_t bucket_bytes(const BucketParams& p) { return (2 * static_cast<size_t>(p.R) + 1) * sizeof(uint16_t); }

// Threads of a backward workgroup: as many columns as 64 KiB of LDS hold (two workgroups a CU), in whole
// waves, and with the heads innermost at least one for each head.
int bwd_threads(const BucketParams& p) {
  const int least = p.qkh ? (p.H + 63) / 64 * 64 : 64;
  int t = kThreads;
  while (t > least && (static_cast<size_t>(p.nb) + 1) * t * sizeof(float) > (64u << 10)) t -= 64;
  return t;
}

int bwd_slots(const BucketParams& p) {
  const int T = bwd_threads(p), heads = p.qkh ? p.H : 1, pairs = T / heads;
  const int64_t n = (p.B * p.Nq * p.Nk + pairs - 1) / pairs, most = p.qkh ? 1024 : (1024 + p.H - 1) / p.H;
  return static_cast<int>(n < most ? n : most);
}

template <class K>
hipError_t allow_lds(K kernel, size_t bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes));
}

template <class S, bool QKH>
hipError_t run_bwd(const BucketParams& p, const void* de, float* partial, hipStream_t stream) {
  const int T = bwd_threads(p);
  const size_t lds = (static_cast<size_t>(p.nb) + 1) * T * sizeof(float) + bucket_bytes(p);
  if (hipError_t err = allow_lds(bucket_bias_bwd_kernel<S, QKH>, lds); err != hipSuccess) return err;
  bucket_bias_bwd_kernel<S, QKH><<<dim3(bwd_slots(p), QKH ? 1 : p.H), T, lds, stream>>>(p, de, partial);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_bucket_bias_fwd(const BucketParams& p, const float* table, void* e, hipStream_t stream) {
  const size_t lds = (static_cast<size_t>(p.nb) + 1) * p.H * sizeof(float) + bucket_bytes(p);
  const int64_t items = p.B * p.Nq * p.Nk * (p.qkh ? p.H : 1), n = (items + kThreads - 1) / kThreads;
  const unsigned grid = static_cast<unsigned>(n < 4096 ? n : 4096);
  auto go = [&](auto kernel) {
    if (hipError_t err = allow_lds(kernel, lds); err != hipSuccess) return err;
    kernel<<<grid, kThreads, lds, stream>>>(p, table, e);
    return hipGetLastError();
  };
  const bool bf16 = p.dtype == HZ_DTYPE_BF16;
  if (p.qkh) return bf16 ? go(bucket_bias_qkh_kernel<BF16>) : go(bucket_bias_qkh_kernel<F32>);
  return bf16 ? go(bucket_bias_qhk_kernel<BF16>) : go(bucket_bias_qhk_kernel<F32>);
}

int64_t bucket_bias_workspace(const BucketParams& p) {
  return static_cast<int64_t>(bwd_slots(p)) * p.nb * p.H * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_bucket_bias_bwd(const BucketParams& p, const void* de, float* dtable, void* workspace,
                                  hipStream_t stream) {
  float* const partial = static_cast<float*>(workspace);
  const bool bf16 = p.dtype == HZ_DTYPE_BF16;
  const hipError_t err = p.qkh ? (bf16 ? run_bwd<BF16, true>(p, de, partial, stream) : run_bwd<F32, true>(p, de, partial, stream))
                               : (bf16 ? run_bwd<BF16, false>(p, de, partial, stream) : run_bwd<F32, false>(p, de, partial, stream));
  if (err != hipSuccess) return err;
  const int n = p.nb * p.H;
  bucket_sum_kernel<<<(n + 15) / 16, kThreads, 0, stream>>>(partial, bwd_slots(p), n, dtable);
  return hipGetLastError();
}

}  // namespace hz
