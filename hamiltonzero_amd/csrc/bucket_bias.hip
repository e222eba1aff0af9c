// Learned relative position bias by buckets, written into the attention's bias layouts, and its
// table's gradient (formulas: include/hz_token.h).
//
// Forward: one lookup in LDS an element; bound by the bytes it writes.
// Backward: a histogram of de by bucket, in one of two ways.
// [B, Nq, H, Nk]: a workgroup stays on one head and every thread adds its elements to a column of its own in LDS
// (bank = lane: no conflicts; plain reads and writes, since LDS's float atomics take 200 cycles a wave).
// [B, Nq, Nk, H]: the pairs of query and key share their bucket among all heads, so the histogram is a product,
// dtable = onehot(bucket)^T de, on the bfloat16 matrix cores: zeros and ones are exact, float32 gradients go in three
// parts whose sum they are (split_f32.h), and the sums are float32.
// Either way a second kernel sums the workgroups' rows: one order of additions, whatever the order in which
// workgroups run. Bound by the bytes it reads (bias_train_sites_f32's 134 MB: 29 us, 4.6 TB/s).
#include "mhsea_device.h"
#include "split_f32.h"
#include "token_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;

// Row of `buckets` in LDS for a pair's distance; the subtraction saturates, so any two positions have one.
__device__ __forceinline__ int bucket_of(const BucketParams& p, const uint16_t* buckets, int qpos, int kpos) {
  const int d = __builtin_elementwise_sub_sat(kpos, qpos);
  return buckets[p.R + min(max(d, -p.R), p.R)];
}

// buckets to LDS; a number outside the table becomes nb, a bucket whose bias is zero.
__device__ __forceinline__ void stage_buckets(const BucketParams& p, uint16_t* buckets, int threads) {
  for (int i = threadIdx.x; i < 2 * p.R + 1; i += threads) {
    const int m = p.buckets[i];
    buckets[i] = static_cast<uint16_t>(m < 0 || m >= p.nb ? p.nb : m);
  }
}

// V consecutive elements in storage format.
template <class S, int V>
struct alignas(V * S::kBytes) Pack {
  typename S::T x[V];
};

__device__ __forceinline__ void put(float v, float& x) { x = v; }
__device__ __forceinline__ void put(float v, uint16_t& x) { x = f32_to_bf16(v); }
__device__ __forceinline__ float get(float x) { return x; }
__device__ __forceinline__ float get(uint16_t x) { return bf16_to_f32(x); }

// How a workgroup's T threads lie over the pairs of query and key (their V-element packs): `across` of them on
// one row of keys, the others on the following rows.
struct Lay {
  int across, rows, x, row;  // this thread's place; row >= rows: idle
  __device__ __forceinline__ Lay(int T, int width) {
    across = width < T ? width : T;
    rows = T / across;
    row = threadIdx.x / across;
    x = threadIdx.x - row * across;
  }
};

// [B, Nq, H, Nk]: a thread takes V keys of a query and writes them for every head.
template <class S, int V>
__global__ void __launch_bounds__(kThreads) bucket_bias_qhk_kernel(BucketParams p, const float* table, void* e) {
  extern __shared__ float lds[];
  const int ld = p.nb + 1;  // a row of buckets for each head
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + p.H * ld);
  for (int i = threadIdx.x; i < p.H * ld; i += kThreads) {
    const int h = i / ld, m = i - h * ld;
    lds[i] = m < p.nb ? table[static_cast<int64_t>(m) * p.H + h] : 0.f;
  }
  stage_buckets(p, buckets, kThreads);
  __syncthreads();
  const int rows = static_cast<int>(p.B * p.Nq), Nk = static_cast<int>(p.Nk), width = Nk / V;
  const Lay lay(kThreads, width);
  if (lay.row >= lay.rows) return;
  typename S::T* const out = static_cast<typename S::T*>(e);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * lay.rows + lay.row; row < rows;
       row += static_cast<int64_t>(gridDim.x) * lay.rows) {
    const int b = static_cast<int>(row) / static_cast<int>(p.Nq), qpos = p.qpos[row];
    const int32_t* const kpos = p.kpos + static_cast<int64_t>(b) * Nk;
    for (int x = lay.x; x < width; x += lay.across) {
      int m[V];
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = bucket_of(p, buckets, qpos, kpos[x * V + v]);
      typename S::T* to = out + row * p.H * Nk + x * V;
#pragma unroll 4
      for (int h = 0; h < p.H; ++h, to += Nk) {
        Pack<S, V> y;
#pragma unroll
        for (int v = 0; v < V; ++v) put(lds[h * ld + m[v]], y.x[v]);
        if constexpr (V == 1)
          *to = y.x[0];
        else
          *reinterpret_cast<uint32_t*>(to) = __builtin_bit_cast(uint32_t, y);
      }
    }
  }
}

// [B, Nq, Nk, H]: a thread takes V heads of a pair; the table lies in LDS as it is written. V elements fill
// 16 bytes, or V is 1.
template <class S, int V>
__global__ void __launch_bounds__(kThreads) bucket_bias_qkh_kernel(BucketParams p, const float* table, void* e) {
  extern __shared__ __align__(16) char raw[];
  typedef typename S::T T;
  T* const lds = reinterpret_cast<T*>(raw);
  const int n = p.nb * p.H, all = n + p.H;
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + (all + 1) / 2 * 2);
  for (int i = threadIdx.x; i < all; i += kThreads) put(i < n ? table[i] : 0.f, lds[i]);
  stage_buckets(p, buckets, kThreads);
  __syncthreads();
  const int rows = static_cast<int>(p.B * p.Nq), Nk = static_cast<int>(p.Nk), packs = p.H / V;
  const int pairs = kThreads / packs;  // pairs at a time (H <= 256: at least one)
  const int pair = threadIdx.x / packs, h = (threadIdx.x - pair * packs) * V;
  if (pair >= pairs) return;
  const Lay lay = [&] {
    Lay l(pairs, Nk);
    l.row = pair / l.across;
    l.x = pair - l.row * l.across;
    return l;
  }();
  if (lay.row >= lay.rows) return;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * lay.rows + lay.row; row < rows;
       row += static_cast<int64_t>(gridDim.x) * lay.rows) {
    const int b = static_cast<int>(row) / static_cast<int>(p.Nq), qpos = p.qpos[row];
    const int32_t* const kpos = p.kpos + static_cast<int64_t>(b) * Nk;
    T* const out = static_cast<T*>(e) + row * Nk * p.H + h;
#pragma unroll 4
    for (int j = lay.x; j < Nk; j += lay.across) {
      const T* const from = lds + bucket_of(p, buckets, qpos, kpos[j]) * p.H + h;
      T* const to = out + static_cast<int64_t>(j) * p.H;
      if constexpr (V == 1)
        *to = *from;
      else
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
    }
  }
}

// n / d for n < 2^31 by one multiplication (Granlund and Montgomery, "Division by Invariant Integers using
// Multiplication", 1994: with s = ceil(log2 d) - 1 and m = floor(2^(32 + s) / d) + 1 the error stays below 1).
struct Divider {
  uint32_t m;
  int s, d;
  static Divider of(int d) {
    int s = 0;
    while ((int64_t(2) << s) < d) ++s;
    return {d == 1 ? 0u : static_cast<uint32_t>((uint64_t(1) << (32 + s)) / static_cast<uint64_t>(d) + 1), s, d};
  }
  __device__ __forceinline__ int of_row(int n) const {
    return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> s);
  }
};

// Partial gradients partial [slots][nb][H], grid (slots, H): every thread on head blockIdx.y and V consecutive keys.
template <class S, int V>
__global__ void bucket_bias_bwd_qhk_kernel(BucketParams p, Divider by_nq, const void* de, float* partial) {
  extern __shared__ float lds[];
  constexpr int U = 4;  // packs a thread loads at a time
  const int T = blockDim.x, tid = threadIdx.x, h = blockIdx.y;
  uint16_t* const buckets = reinterpret_cast<uint16_t*>(lds + (p.nb + 1) * T);
  for (int i = tid; i < (p.nb + 1) * T; i += T) lds[i] = 0.f;
  stage_buckets(p, buckets, T);
  __syncthreads();
  const int rows = static_cast<int>(p.B * p.Nq), Nk = static_cast<int>(p.Nk), width = Nk / V;
  const Lay lay(T, width);
  typedef Pack<S, V> P;
  if (lay.row < lay.rows) {
    float* const mine = lds + tid;
    const int64_t step = static_cast<int64_t>(gridDim.x) * lay.rows;
    int64_t row = static_cast<int64_t>(blockIdx.x) * lay.rows + lay.row;
    int x = lay.x;
    while (row < rows) {
      // U packs, all loads first and without branches: what lies behind the last row is the last pack again and
      // goes into the bucket that is not summed
      P g[U];
      int at[U * V], m[U * V], qp[U];
      bool on[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        on[u] = row < rows;
        const int r = static_cast<int>(on[u] ? row : rows - 1);
        qp[u] = p.qpos[r];
        const int32_t* const kpos = p.kpos + static_cast<int64_t>(by_nq.of_row(r)) * Nk + x * V;
#pragma unroll
        for (int v = 0; v < V; ++v) at[u * V + v] = kpos[v];
        g[u] = *reinterpret_cast<const P*>(static_cast<const typename S::T*>(de) + (static_cast<int64_t>(r) * p.H + h) * Nk + x * V);
        x += lay.across;
        row += x < width ? 0 : step;
        x = x < width ? x : lay.x;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int bucket = bucket_of(p, buckets, qp[u], at[u * V + v]);
          m[u * V + v] = (on[u] ? bucket : p.nb) * T;
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) mine[m[u * V + v]] += get(g[u].x[v]);
    }
  }
  __syncthreads();
  // the workgroup's sums: a wave a bucket, its threads' columns in a fixed order
  for (int m = tid >> 6; m < p.nb; m += T >> 6) {
    float sum = 0.f;
    for (int t = tid & 63; t < T; t += 64) sum += lds[m * T + t];
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
    if ((tid & 63) == 0) partial[(static_cast<int64_t>(blockIdx.x) * p.nb + m) * p.H + h] = sum;
  }
}

constexpr int kBlocks = 4;  // blocks of 16 buckets a workgroup of the product has sums for

// Partial gradients partial [slots][nb][H], grid (slots, groups of 16 HB heads, groups of 64 buckets): four waves
// on 64 consecutive pairs of query and key at a time, each in LDS of its own (no barriers). Operands
// (v_mfma_f32_16x16x32_bf16, split_f32.h): A = one-hot rows of buckets, B = de, both over the pairs
// 16 (j / 4) + 4 g + j % 4 of 32, the order in which transposing reads of de's rows come without bank
// conflicts. WIDE: heads in 16-byte chunks, else one by one.
template <class S, int HB, bool WIDE>
__global__ void __launch_bounds__(kThreads) bucket_bias_bwd_qkh_kernel(BucketParams p, Divider by_nk, Divider by_nq,
                                                                       int rows_each, const void* de, float* partial) {
  constexpr int PARTS = S::kBytes == 4 ? 3 : 1;
  constexpr int E = WIDE ? 16 / S::kBytes : 1;  // elements a chunk
  constexpr int PER = 16 * HB / E;              // chunks a pair
  typedef short v4s __attribute__((ext_vector_type(4)));
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  __shared__ __align__(16) uint16_t tiles[4][HB][PARTS][64][16];
  __shared__ __align__(16) uint16_t numbers[4][64];
  extern __shared__ uint16_t buckets[];
  stage_buckets(p, buckets, kThreads);
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int h0 = blockIdx.y * 16 * HB, m0 = blockIdx.z * 16 * kBlocks, Nk = static_cast<int>(p.Nk);
  const int64_t rows = p.B * p.Nq;
  v4f acc[kBlocks][HB];
#pragma unroll
  for (int m = 0; m < kBlocks; ++m)
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) acc[m][hb] = zero4();

  typedef std::conditional_t<WIDE, v4u, typename S::T> Chunk;
  for (int64_t row0 = 0; row0 < rows; row0 += rows_each) {  // pairs of one round are numbered in 31 bits
    const int total = static_cast<int>((rows - row0 < rows_each ? rows - row0 : rows_each) * Nk);
    const typename S::T* const from = static_cast<const typename S::T*>(de) + row0 * Nk * p.H + h0;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
    Chunk x[PER];
    int qpos = 0, kpos = 0;
    auto load = [&](int64_t f0) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int q = u * 64 + lane, pair = q / PER, part = q % PER;
        x[u] = Chunk{};
        if (f0 + pair < total && h0 + part * E < p.H) x[u] = *reinterpret_cast<const Chunk*>(from + (f0 + pair) * p.H + part * E);
      }
      const int f = static_cast<int>(f0 + lane < total ? f0 + lane : total - 1), r = by_nk.of_row(f), j = f - r * Nk;
      const int row = static_cast<int>(row0) + r;
      qpos = p.qpos[row];
      kpos = p.kpos[static_cast<int64_t>(by_nq.of_row(row)) * Nk + j];
    };
    int64_t f0 = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * 64;
    if (f0 < total) load(f0);
    for (; f0 < total; f0 += stride) {
      numbers[wave][lane] = static_cast<uint16_t>(f0 + lane < total ? bucket_of(p, buckets, qpos, kpos) : 0xffff);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int q = u * 64 + lane, pair = q / PER, col = q % PER * E;
        uint16_t* const to = &tiles[wave][col / 16][0][pair][col % 16];
        if constexpr (PARTS == 1) {
          *reinterpret_cast<Chunk*>(to) = x[u];
        } else if constexpr (WIDE) {
          uint32_t w[2][3];
          split2(__uint_as_float(x[u][0]), __uint_as_float(x[u][1]), w[0][0], w[0][1], w[0][2]);
          split2(__uint_as_float(x[u][2]), __uint_as_float(x[u][3]), w[1][0], w[1][1], w[1][2]);
#pragma unroll
          for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(to + i * 64 * 16) = make_uint2(w[0][i], w[1][i]);
        } else {
          uint32_t w[3];
          split2(x[u], 0.f, w[0], w[1], w[2]);
#pragma unroll
          for (int i = 0; i < 3; ++i) to[i * 64 * 16] = static_cast<uint16_t>(w[i]);
        }
      }
      if (f0 + stride < total) load(f0 + stride);  // in flight during the products
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v4u b[HB][PARTS];
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            uint16_t* const at = &tiles[wave][hb][i][32 * k + 4 * g + (c >> 2)][4 * (c & 3)];
            const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at));
            const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at + 16 * 16));
            const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
            b[hb][i] = v4u{l.x, l.y, h.x, h.y};
          }
        const uint2 n0 = *reinterpret_cast<const uint2*>(&numbers[wave][32 * k + 4 * g]);
        const uint2 n1 = *reinterpret_cast<const uint2*>(&numbers[wave][32 * k + 16 + 4 * g]);
        const uint32_t n[4] = {n0.x, n0.y, n1.x, n1.y};
#pragma unroll
        for (int m = 0; m < kBlocks; ++m) {
          if (m0 + 16 * m >= p.nb) break;
          const uint16_t target = static_cast<uint16_t>(m0 + 16 * m + c);
          v4u a;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // 1.0 where the pair's number is the row's, else 0
            const u16x2 off = __builtin_bit_cast(u16x2, n[i]) ^ u16x2{target, target};
            a[i] = __builtin_bit_cast(uint32_t, (u16x2{1, 1} - __builtin_elementwise_min(off, u16x2{1, 1})) * u16x2{0x3f80, 0x3f80});
          }
#pragma unroll
          for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int i = PARTS - 1; i >= 0; --i) acc[m][hb] = mfma16_bf16(as_bf16x8(a), as_bf16x8(b[hb][i]), acc[m][hb]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
  // the four waves' sums, one after the other
  __syncthreads();
  float* const red = reinterpret_cast<float*>(tiles);  // [wave][16][16]
  for (int m = 0; m < kBlocks && m0 + 16 * m < p.nb; ++m)
    for (int hb = 0; hb < HB; ++hb) {
      v4f mine = acc[0][0];
#pragma unroll
      for (int mm = 0; mm < kBlocks; ++mm)
#pragma unroll
        for (int hh = 0; hh < HB; ++hh) mine = mm == m && hh == hb ? acc[mm][hh] : mine;
#pragma unroll
      for (int r = 0; r < 4; ++r) red[(wave * 16 + 4 * g + r) * 16 + c] = mine[r];
      __syncthreads();
      const int i = threadIdx.x, row = m0 + 16 * m + i / 16, col = h0 + 16 * hb + i % 16;
      const float sum = (red[i] + red[256 + i]) + (red[512 + i] + red[768 + i]);
      if (row < p.nb && col < p.H) partial[(static_cast<int64_t>(blockIdx.x) * p.nb + row) * p.H + col] = sum;
      __syncthreads();
    }
}

__global__ void __launch_bounds__(kThreads) bucket_sum_kernel(const float* partial, int slots, int n, float* dtable) {
  __shared__ float red[kThreads];
  const int c = threadIdx.x % 16, r0 = threadIdx.x / 16, col = blockIdx.x * 16 + c;
  float sum = 0.f;
  if (col < n)
#pragma unroll 8
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

// [B, Nq, H, Nk]: threads of a workgroup, as many as 64 KiB of LDS hold columns of (two workgroups a CU), in whole
// waves.
int qhk_threads(const BucketParams& p) {
  int t = kThreads;
  while (t > 64 && (static_cast<size_t>(p.nb) + 1) * t * sizeof(float) > (64u << 10)) t -= 64;
  return t;
}
bool qhk_wide(const BucketParams& p) { return p.Nk % 4 == 0; }

// [B, Nq, Nk, H]: blocks of 16 heads a workgroup: three parts of two fill 48 KiB of LDS, and heads one by one take a
// register each for 64 pairs.
int qkh_blocks(const BucketParams& p) {
  return p.H <= 16 ? 1 : p.H <= 32 || p.dtype == HZ_DTYPE_F32 || p.H % 8 != 0 ? 2 : 4;
}

// Workgroups over the pairs: 1024 in all, with some work for each.
int bwd_slots(const BucketParams& p) {
  const int64_t pairs = p.B * p.Nq * p.Nk;
  int64_t n, most;
  if (p.qkh) {
    n = pairs / 512;
    most = 1024;
  } else {
    n = pairs / (qhk_wide(p) ? 4 : 1) / (qhk_threads(p) * 8);
    most = (1024 + p.H - 1) / p.H;
  }
  return static_cast<int>(n < 1 ? 1 : n < most ? n : most);
}

// The most dynamic LDS a kernel is launched with: a limit of the function's, so every call sets the same one, and calls of
// other sizes in other threads do not lower it between this and the launch.
constexpr size_t kMostBuckets = (2 * HZ_BUCKET_MAX_RANGE + 1) * sizeof(uint16_t);
constexpr size_t kMostTable = HZ_BUCKET_MAX_TABLE * sizeof(float);  // (n_buckets + 1) rows of H, or of 64 threads
static_assert((HZ_BUCKET_MAX + 1) * 64 <= HZ_BUCKET_MAX_TABLE && kMostTable + kMostBuckets <= (160u << 10));
template <class K>
hipError_t allow_lds(K kernel, size_t most) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(most));
}

template <class S, int V>
hipError_t run_qhk(const BucketParams& p, const void* de, float* partial, hipStream_t stream) {
  const int T = qhk_threads(p);
  const size_t lds = (static_cast<size_t>(p.nb) + 1) * T * sizeof(float) + bucket_bytes(p);
  if (hipError_t err = allow_lds(bucket_bias_bwd_qhk_kernel<S, V>, kMostTable + kMostBuckets); err != hipSuccess) return err;
  bucket_bias_bwd_qhk_kernel<S, V><<<dim3(bwd_slots(p), p.H), T, lds, stream>>>(p, Divider::of(static_cast<int>(p.Nq)), de, partial);
  return hipGetLastError();
}

template <class S, int HB, bool WIDE>
hipError_t run_qkh(const BucketParams& p, const void* de, float* partial, hipStream_t stream) {
  if (hipError_t err = allow_lds(bucket_bias_bwd_qkh_kernel<S, HB, WIDE>, kMostBuckets); err != hipSuccess) return err;
  const dim3 grid(bwd_slots(p), (p.H + 16 * HB - 1) / (16 * HB), (p.nb + 16 * kBlocks - 1) / (16 * kBlocks));
  const int64_t rows = p.B * p.Nq, most = (int64_t(1) << 30) / p.Nk, each = most < 1 ? 1 : most < rows ? most : rows;
  bucket_bias_bwd_qkh_kernel<S, HB, WIDE><<<grid, kThreads, bucket_bytes(p), stream>>>(
      p, Divider::of(static_cast<int>(p.Nk)), Divider::of(static_cast<int>(p.Nq)), static_cast<int>(each), de, partial);
  return hipGetLastError();
}

template <class S, int HB>
hipError_t run_qkh(const BucketParams& p, const void* de, float* partial, hipStream_t stream) {
  if constexpr (HB < 4)
    if (p.H % (16 / S::kBytes) != 0) return run_qkh<S, HB, false>(p, de, partial, stream);
  return run_qkh<S, HB, true>(p, de, partial, stream);
}

}  // namespace

hipError_t launch_bucket_bias_fwd(const BucketParams& p, const float* table, void* e, hipStream_t stream) {
  const bool bf16 = p.dtype == HZ_DTYPE_BF16;
  const int64_t elements = p.B * p.Nq * p.Nk * p.H, n = elements / (kThreads * 16) + 1;
  const unsigned grid = static_cast<unsigned>(n < 2048 ? n : 2048);
  auto go = [&](auto kernel, size_t table_bytes) {
    const size_t lds = table_bytes + bucket_bytes(p);
    if (hipError_t err = allow_lds(kernel, kMostTable + kMostBuckets); err != hipSuccess) return err;
    kernel<<<grid, kThreads, lds, stream>>>(p, table, e);
    return hipGetLastError();
  };
  const size_t entries = (static_cast<size_t>(p.nb) + 1) * p.H;
  if (p.qkh) {
    const size_t bytes = (entries + 1) / 2 * 2 * (bf16 ? 2 : 4);
    if (bf16) return p.H % 8 == 0 ? go(bucket_bias_qkh_kernel<BF16, 8>, bytes) : go(bucket_bias_qkh_kernel<BF16, 1>, bytes);
    return p.H % 4 == 0 ? go(bucket_bias_qkh_kernel<F32, 4>, bytes) : go(bucket_bias_qkh_kernel<F32, 1>, bytes);
  }
  if (bf16 && p.Nk % 2 == 0) return go(bucket_bias_qhk_kernel<BF16, 2>, entries * 4);
  return bf16 ? go(bucket_bias_qhk_kernel<BF16, 1>, entries * 4) : go(bucket_bias_qhk_kernel<F32, 1>, entries * 4);
}

int64_t bucket_bias_workspace(const BucketParams& p) {
  return static_cast<int64_t>(bwd_slots(p)) * p.nb * p.H * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_bucket_bias_bwd(const BucketParams& p, const void* de, float* dtable, void* workspace,
                                  hipStream_t stream) {
  float* const partial = static_cast<float*>(workspace);
  const bool f32 = p.dtype == HZ_DTYPE_F32, wide = qhk_wide(p);
  const int blocks = qkh_blocks(p);
  hipError_t err;
  if (!p.qkh && f32)
    err = wide ? run_qhk<F32, 4>(p, de, partial, stream) : run_qhk<F32, 1>(p, de, partial, stream);
  else if (!p.qkh)
    err = wide ? run_qhk<BF16, 4>(p, de, partial, stream) : run_qhk<BF16, 1>(p, de, partial, stream);
  else if (f32)
    err = blocks == 1 ? run_qkh<F32, 1>(p, de, partial, stream) : run_qkh<F32, 2>(p, de, partial, stream);
  else
    err = blocks == 1   ? run_qkh<BF16, 1>(p, de, partial, stream)
          : blocks == 2 ? run_qkh<BF16, 2>(p, de, partial, stream)
                        : run_qkh<BF16, 4>(p, de, partial, stream);
  if (err != hipSuccess) return err;
  const int n = p.nb * p.H;
  bucket_sum_kernel<<<(n + 15) / 16, kThreads, 0, stream>>>(partial, bwd_slots(p), n, dtable);
  return hipGetLastError();
}

}  // namespace hz
