// Paged caches: new tokens into their slots, and eviction by accumulated weight (include/hz_paged.h).
//
// Append: a thread copies 16 bytes of a key or value; bound by those bytes.
//
// Eviction, of each row and key head: the smallest score that stays, the places of the slots given up below the budget
// (holes) and of the kept ones behind it, and the moves of the k-th of these into the k-th of those.
// Sources lie behind the budget and targets below it, so the moves do not depend on each other, and what
// stays below is not touched: about budget (1 - budget / n) tokens are read and written and not the whole
// budget, which a compaction in order would move.
//   Up to 1024 slots, one wave has a row in its registers and finds the score bit by bit from the top by counting; then all waves of
// its workgroup move the tokens. More slots are a workgroup's of 16 waves, up to 32768 in registers: the
// score by its top 11, next 11 and last 10 bits with a histogram in LDS for each; then each thread counts its
// holes and late slots, and one scan gives them their numbers. A second kernel, with workgroups enough for all of
// them, moves the tokens.
#include "mhsea_device.h"
#include "paged_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads) paged_append_kernel(Pages c, hz_token_tensor k, hz_token_tensor v, int64_t total, int N,
                                                                int Hk, int chunks, int bytes) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= total) return;
  const int ch = static_cast<int>(id % chunks);
  int64_t r = id / chunks;
  const int h = static_cast<int>(r % Hk);
  r /= Hk;
  const int i = static_cast<int>(r % N), b = static_cast<int>(r / N);
  const int slot = c.length(b) - N + i;
  if (slot < 0) return;
  const int at = c.page_of(slot), page = c.table[static_cast<int64_t>(b) * c.width + at], in = slot - at * c.size;
  if (page < 0 || page >= c.pages) return;
  const int64_t from_k = b * k.batch + i * k.token + h * k.head, from_v = b * v.batch + i * v.token + h * v.head;
  const int64_t to_k = page * c.page_k + in * c.token_k + h * c.head_k, to_v = page * c.page_v + in * c.token_v + h * c.head_v;
  const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const char*>(k.data) + from_k * bytes + 16 * ch);
  const uint4 y = *reinterpret_cast<const uint4*>(static_cast<const char*>(v.data) + from_v * bytes + 16 * ch);
  *reinterpret_cast<uint4*>(static_cast<char*>(const_cast<void*>(c.k)) + to_k * bytes + 16 * ch) = x;
  *reinterpret_cast<uint4*>(static_cast<char*>(const_cast<void*>(c.v)) + to_v * bytes + 16 * ch) = y;
}

// --- eviction -----------------------------------------------------------------------------------------------------------

constexpr int kSelect = 1024;  // threads of a long row's workgroup
constexpr int kWaves = kSelect / 64;
constexpr int kWaveSlots = 1024;  // most slots of a row that one wave cuts

struct EvictParams {
  Pages c;
  const float* scores;
  float* scores_out;
  int32_t *sources, *lengths_out;
  int32_t *count, *from, *to;  // of each row and key head: its moves
  int B, Hk, budget, keep, sinks, recent, most;  // keep: min(budget, slots); most: moves at most
  int chunks, bytes;                             // 16-byte chunks of a head; bytes of an element
};

// The order of scores as unsigned numbers, all below kFixed; NaN is the least, -0 equals 0.
constexpr uint32_t kFixed = 0xffffffffu;
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

// (A signed number: the hardware's count is unsigned, and what is compared with it may be negative.)
__device__ __forceinline__ int bits(uint64_t votes) { return static_cast<int>(__popcll(votes)); }

// One row and key head: of its n slots m stay, those below lo and from hi on whatever their scores.
struct Row {
  int64_t row;
  int b, h, n, m, lo, hi;
  const float* scores;
  float* scores_out;
  int32_t* sources;
  __device__ __forceinline__ Row(const EvictParams& p, int64_t row_) : row(row_), b(static_cast<int>(row_ / p.Hk)), h(static_cast<int>(row_ % p.Hk)) {
    n = p.c.length(b), m = p.budget, lo = p.sinks, hi = n - p.recent;
    scores = p.scores + row * p.c.slots;
    scores_out = p.scores_out + row * p.c.slots;
    sources = p.sources + row * p.keep;
  }
  // What does not depend on the scores, and the slots below the budget as if all of them stayed, by `threads` threads. (Loads are
  // unconditional, so that none waits for another; 16 bytes at a time where rows are a multiple of four slots.)
  __device__ __forceinline__ void fill(const EvictParams& p, int tid, int threads) const {
    if (tid == 0 && h == 0) p.lengths_out[b] = min(n, m);
    const int end = min(n, m);
    if (p.c.slots % 4 == 0) {
#pragma unroll 4
      for (int s = 4 * tid; s < p.c.slots; s += 4 * threads) {
        float4 x = *reinterpret_cast<const float4*>(scores + min(s, (m - 1) & ~3));
        x.x = s < end ? x.x : 0.f, x.y = s + 1 < end ? x.y : 0.f, x.z = s + 2 < end ? x.z : 0.f, x.w = s + 3 < end ? x.w : 0.f;
        *reinterpret_cast<float4*>(scores_out + s) = x;
      }
    } else {
#pragma unroll 4
      for (int s = tid; s < p.c.slots; s += threads) {
        const float x = scores[min(s, m - 1)];
        scores_out[s] = s < end ? x : 0.f;
      }
    }
#pragma unroll 4
    for (int s = tid; s < p.keep; s += threads) sources[s] = s < n ? s : -1;
  }
  // The key of slot s, whose score is x; 0 behind the row.
  __device__ __forceinline__ uint32_t key(int s, float x) const { return s >= n ? 0u : s >= lo && s < hi ? ordered(x) : kFixed; }
  // A lane's keys of the slots base + step j.
  template <int KEYS>
  __device__ __forceinline__ void keys(int base, int step, uint32_t (&u)[KEYS]) const {
    float x[KEYS];
#pragma unroll
    for (int j = 0; j < KEYS; ++j) x[j] = scores[min(base + step * j, n - 1)];
#pragma unroll
    for (int j = 0; j < KEYS; ++j) u[j] = key(base + step * j, x[j]);
  }
  // Of the slots base + j, where rows are a multiple of four slots and base is one.
  template <int KEYS>
  __device__ __forceinline__ void keys_by_four(int base, uint32_t (&u)[KEYS]) const {
    float4 x[KEYS / 4];
#pragma unroll
    for (int j = 0; j < KEYS / 4; ++j) x[j] = *reinterpret_cast<const float4*>(scores + min(base + 4 * j, (n - 1) & ~3));
#pragma unroll
    for (int j = 0; j < KEYS / 4; ++j) {
      const int s = base + 4 * j;
      u[4 * j] = key(s, x[j].x), u[4 * j + 1] = key(s + 1, x[j].y), u[4 * j + 2] = key(s + 2, x[j].z), u[4 * j + 3] = key(s + 3, x[j].w);
    }
  }
};

// A wave's slots 64 j + lane < n, with their keys, to the lists: slots below the budget that go (holes) and slots behind it that stay
// (late), in ascending order. Slots above the threshold stay, and `equal` at it. Returns the number of holes, which is that of late slots.
template <int KEYS>
__device__ __forceinline__ int put_moves(const Row& r, uint32_t threshold, int equal, const uint32_t (&u)[KEYS], int* to, int* from) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  int holes = 0, late = 0;
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int s0 = 64 * j, s = s0 + lane;
    if (s0 >= r.n) break;
    const bool in = s < r.n;
    bool stays = in && u[j] > threshold;
    const uint64_t votes = __ballot(in && u[j] == threshold);
    if (votes != 0) {
      stays = stays || (in && u[j] == threshold && bits(votes & below) < equal);
      equal -= bits(votes);
    }
    if (s0 < r.m) {
      const bool is = in && s < r.m && !stays;
      const uint64_t v = __ballot(is);
      if (is) to[holes + bits(v & below)] = s;
      holes += bits(v);
    }
    if (s0 + 63 >= r.m) {
      const bool is = s >= r.m && stays;
      const uint64_t v = __ballot(is);
      if (is) from[late + bits(v & below)] = s;
      late += bits(v);
    }
  }
  return holes;
}

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(static_cast<int>(wave_scan(x)), 63); }

// Moves `count` tokens of one row and key head from the slots from[i] to the slots to[i], by `threads` threads: four in flight
// for each group of `chunks` lanes.
template <class List>
__device__ __forceinline__ void move(const EvictParams& p, int b, int h, List from, List to, int begin, int end, int tid, int threads) {
  typedef unsigned v4 __attribute__((ext_vector_type(4)));
  const int32_t* const table = p.c.table + static_cast<int64_t>(b) * p.c.width;
  const int rows = threads / p.chunks, ch = tid % p.chunks, mine = tid / p.chunks;
  if (mine >= rows) return;
  char* const k = static_cast<char*>(const_cast<void*>(p.c.k)) + h * p.c.head_k * p.bytes + 16 * ch;
  char* const v = static_cast<char*>(const_cast<void*>(p.c.v)) + h * p.c.head_v * p.bytes + 16 * ch;
  constexpr int U = 4;
  for (int i0 = begin + mine; i0 < end; i0 += U * rows) {
    int at[U], to_slot[U], page_a[U], page_t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * rows, end - 1);
      at[u] = from[i], to_slot[u] = to[i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) page_a[u] = table[p.c.page_of(at[u])], page_t[u] = table[p.c.page_of(to_slot[u])];
    v4 x[U], y[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      on[u] = i0 + u * rows < end && page_a[u] >= 0 && page_a[u] < p.c.pages && page_t[u] >= 0 && page_t[u] < p.c.pages;
      if (!on[u]) continue;
      const int64_t in = at[u] - p.c.page_of(at[u]) * p.c.size;
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(k + (page_a[u] * p.c.page_k + in * p.c.token_k) * p.bytes));
      y[u] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(v + (page_a[u] * p.c.page_v + in * p.c.token_v) * p.bytes));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) continue;
      const int64_t in = to_slot[u] - p.c.page_of(to_slot[u]) * p.c.size;
      *reinterpret_cast<v4*>(k + (page_t[u] * p.c.page_k + in * p.c.token_k) * p.bytes) = x[u];
      *reinterpret_cast<v4*>(v + (page_t[u] * p.c.page_v + in * p.c.token_v) * p.bytes) = y[u];
    }
  }
}

// A row of up to 64 KEYS slots a workgroup: wave 0 cuts it, all move.
template <int KEYS, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_cut_kernel(EvictParams p) {
  __shared__ int to[32 * KEYS], from[32 * KEYS], moves;  // holes and late slots: at most half of the slots each
  const int tid = threadIdx.x, lane = tid & 63;
  const Row r(p, blockIdx.x);
  if (tid >= 64 || r.n <= r.m) r.fill(p, tid, THREADS);
  if (r.n <= r.m) return;
  if (tid < 64) {
    uint32_t u[KEYS];
    r.keys(lane, 64, u);
    r.fill(p, tid, THREADS);
    // bit by bit: the largest threshold that at least m slots reach, or one that exactly m exceed
    uint32_t threshold = 0;
    for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1) {
      int reach = 0;
      if constexpr (KEYS <= 4) {  // a scalar count a key: 20.2 -> 19.6 us for 2048 rows of four keys a lane, 10.0 -> 11.1 for 32 of sixteen
#pragma unroll
        for (int j = 0; j < KEYS; ++j) reach += bits(__ballot(u[j] >= (threshold | bit)));
      } else {
#pragma unroll
        for (int j = 0; j < KEYS; ++j) reach += u[j] >= (threshold | bit) ? 1 : 0;
        reach = wave_sum(reach);
      }
      if (reach >= r.m) threshold |= bit;
      if (reach == r.m) {
        --threshold;
        break;
      }
    }
    int above = 0;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) above += u[j] > threshold ? 1 : 0;
    const int holes = put_moves(r, threshold, r.m - wave_sum(above), u, to, from);
    if (lane == 0) moves = holes;
  }
  __syncthreads();
  const int count = moves;
  for (int i = tid; i < count; i += THREADS) {
    const int s = to[i], at = from[i];
    r.sources[s] = at;
    r.scores_out[s] = r.scores[at];
  }
  move(p, r.b, r.h, from, to, 0, count, tid, THREADS);
}

// Sum over the workgroup's threads before this one; total: over all.
__device__ __forceinline__ uint32_t before_thread(uint32_t mine, uint32_t* lds, uint32_t& total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t upto = wave_scan(mine);
  __syncthreads();
  if (lane == 63) lds[wave] = upto;
  __syncthreads();
  uint32_t sum = upto - mine;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) sum += lds[w];
    total += lds[w];
  }
  return sum;
}

__device__ __forceinline__ int sum4(const int* x) {
  const int4 v = *reinterpret_cast<const int4*>(x);
  return v.x + v.y + v.z + v.w;
}

// A workgroup a row. A thread has KEYS slots that follow each other, so that ranks are counted in a thread and scanned once. ONE: the
// row's slots are at most 1024 KEYS; else they are taken that many at a time, and read again for every pass.
template <int KEYS, bool ONE>
__global__ void __launch_bounds__(kSelect) paged_select_kernel(EvictParams p) {
  // (four copies of the histogram: lanes that add to one bin wait for each other, and scores share their top bits)
  constexpr int BINS = 2048, SPAN = KEYS * kSelect;
  __shared__ __align__(16) int hist[BINS][4];
  __shared__ uint16_t list[SPAN];  // a span's holes from the front, late slots from the back
  __shared__ uint32_t shared[kWaves];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 63;
  const Row r(p, blockIdx.x);
  if (r.n <= r.m) {
    r.fill(p, tid, kSelect);
    if (tid == 0) p.count[r.row] = 0;
    return;
  }
  uint32_t u[KEYS];
  auto read = [&](int base) {
    if (p.c.slots % 4 == 0)
      r.keys_by_four(base, u);
    else
      r.keys(base, 1, u);
  };
  if (ONE) read(KEYS * tid);
  r.fill(p, tid, kSelect);
  // the threshold: slots above it stay, and the first `equal` of those at it
  uint32_t threshold = 0;
  int equal = r.m;  // still wanted among the slots whose top bits are the threshold's
  for (int top = 32; top > 0;) {  // (ends early where the slots of a bin and above are exactly those wanted)
    const int width = top > 10 ? 11 : 10, shift = top - width;
    *reinterpret_cast<int4*>(hist[tid]) = make_int4(0, 0, 0, 0);
    *reinterpret_cast<int4*>(hist[tid + kSelect]) = make_int4(0, 0, 0, 0);
    __syncthreads();
    for (int s0 = KEYS * tid; s0 < r.n; s0 += SPAN) {
      if (!ONE) read(s0);
#pragma unroll
      for (int j = 0; j < KEYS; ++j)
        if (s0 + j < r.n && (top == 32 || (u[j] ^ threshold) >> top == 0))
          atomicAdd(&hist[u[j] >> shift & ((1u << width) - 1)][lane & 3], 1);
    }
    __syncthreads();
    // sums from the top bin down, two bins a thread
    const int bin = BINS - 1 - 2 * tid, a = sum4(hist[bin]), c = sum4(hist[bin - 1]);
    uint32_t total;
    const int above = static_cast<int>(before_thread(a + c, shared, total));
    if (above < equal && above + a >= equal) found[0] = bin, found[1] = above, found[2] = a;
    if (above + a < equal && above + a + c >= equal) found[0] = bin - 1, found[1] = above + a, found[2] = c;
    __syncthreads();
    threshold |= static_cast<uint32_t>(found[0]) << shift;
    equal -= found[1];
    top = shift;
    if (equal == found[2]) {
      --threshold;  // all of the bin stay, and nothing below it: the bin's lower end less one, which no kept slot is at
      equal = 0;    // (a bin with something below it: its lower end is not 0)
      break;
    }
    __syncthreads();
  }
  int32_t* const from = p.from + r.row * p.most;
  int32_t* const to = p.to + r.row * p.most;
  int holes = 0, late = 0;  // of the spans before
  for (int base = 0; base < r.n; base += SPAN) {
    const int s0 = base + KEYS * tid;
    if (!ONE) read(s0);
    int mine = 0, rank = 0;
    uint32_t total = 0;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) mine += s0 + j < r.n && u[j] == threshold ? 1 : 0;
    if (equal > 0) rank = static_cast<int>(before_thread(mine, shared, total));
    // a bit a slot, so that the second loop has no ranks to count
    uint32_t stays = 0;
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      const bool same = u[j] == threshold;
      if (s0 + j < r.n && (u[j] > threshold || (same && rank < equal))) stays |= 1u << j;
      rank += same ? 1 : 0;
    }
    equal = max(equal - static_cast<int>(total), 0);
    const int in = min(max(r.n - s0, 0), KEYS), near = min(max(r.m - s0, 0), in);  // slots of the row; below the budget
    const uint32_t all = in == 32 ? 0xffffffffu : (1u << in) - 1, low = near == 32 ? 0xffffffffu : (1u << near) - 1;
    uint32_t hole = low & ~stays, behind = all & ~low & stays;
    const uint32_t counts = before_thread(static_cast<uint32_t>(__popc(hole)) | static_cast<uint32_t>(__popc(behind)) << 16, shared, total);
    const int hole_count = total & 0xffff, late_count = total >> 16;
    int at = counts & 0xffff, back = SPAN - 1 - static_cast<int>(counts >> 16);
    while (hole != 0) {
      const int j = __ffs(hole) - 1;
      list[at++] = static_cast<uint16_t>(KEYS * tid + j);
      hole &= hole - 1;
    }
    while (behind != 0) {
      const int j = __ffs(behind) - 1;
      list[back--] = static_cast<uint16_t>(KEYS * tid + j);
      behind &= behind - 1;
    }
    __syncthreads();
    if (ONE) {
#pragma unroll 4
      for (int i = tid; i < hole_count; i += kSelect) {
        const int s = list[i], source = list[SPAN - 1 - i];
        to[i] = s;
        from[i] = source;
        r.sources[s] = source;
        r.scores_out[s] = r.scores[source];
      }
    } else {
      for (int i = tid; i < hole_count; i += kSelect) to[holes + i] = base + list[i];
      for (int i = tid; i < late_count; i += kSelect) from[late + i] = base + list[SPAN - 1 - i];
      __syncthreads();
    }
    holes += hole_count;
    late += late_count;
  }
  if (!ONE) {
#pragma unroll 4
    for (int i = tid; i < holes; i += kSelect) {
      const int s = to[i], source = from[i];
      r.sources[s] = source;
      r.scores_out[s] = r.scores[source];
    }
  }
  if (tid == 0) p.count[r.row] = holes;
}

// The moves that the selection left: `per_block` of one row and key head a workgroup.
__global__ void __launch_bounds__(kThreads) paged_move_kernel(EvictParams p, int per_block) {
  const int64_t row = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
  if (row >= static_cast<int64_t>(p.B) * p.Hk) return;
  const int begin = blockIdx.x * per_block, end = min(p.count[row], begin + per_block);
  if (begin >= end) return;
  move(p, static_cast<int>(row / p.Hk), static_cast<int>(row % p.Hk), p.from + row * p.most, p.to + row * p.most, begin, end, threadIdx.x, kThreads);
}

int bytes_of(int32_t dtype) { return dtype == HZ_DTYPE_BF16 ? 2 : 4; }

// Moves of a row at most: survivors behind the budget, and holes below it.
int64_t most_moves(const hz_paged_evict_args& a) {
  const int64_t slots = a.cache.page_size * a.cache.table_width, late = slots - a.budget;
  return late <= 0 ? 0 : late < a.budget ? late : a.budget;
}

}  // namespace

hipError_t launch_paged_append(const hz_paged_cache& c, const hz_token_tensor& k, const hz_token_tensor& v, int64_t N,
                               hipStream_t stream) {
  const int bytes = bytes_of(c.dtype), chunks = static_cast<int>(c.D) * bytes / 16;
  const int64_t total = c.B * N * c.Hk * chunks;
  paged_append_kernel<<<static_cast<unsigned>((total + kThreads - 1) / kThreads), kThreads, 0, stream>>>(
      Pages(c), k, v, total, static_cast<int>(N), static_cast<int>(c.Hk), chunks, bytes);
  return hipGetLastError();
}

int64_t paged_evict_workspace(const hz_paged_evict_args& a) {
  if (a.cache.page_size * a.cache.table_width <= kWaveSlots) return 0;
  return a.cache.B * a.cache.Hk * (1 + 2 * most_moves(a)) * static_cast<int64_t>(sizeof(int32_t));
}

hipError_t launch_paged_evict(const hz_paged_evict_args& a, void* workspace, hipStream_t stream) {
  const hz_paged_cache& c = a.cache;
  const int64_t rows = c.B * c.Hk, most = most_moves(a), slots = c.page_size * c.table_width;
  const int bytes = bytes_of(c.dtype), chunks = static_cast<int>(c.D) * bytes / 16;
  EvictParams p{Pages(c), a.scores, a.scores_out, a.sources, a.lengths_out, nullptr, nullptr, nullptr,
                static_cast<int>(c.B), static_cast<int>(c.Hk), static_cast<int>(a.budget),
                static_cast<int>(a.budget < slots ? a.budget : slots), static_cast<int>(a.sinks),
                static_cast<int>(a.recent), static_cast<int>(most), chunks, bytes};
  const unsigned groups = static_cast<unsigned>(rows);
  if (slots <= kWaveSlots) {
    if (slots <= 256)
      paged_cut_kernel<4, 256><<<groups, 256, 0, stream>>>(p);
    else
      paged_cut_kernel<kWaveSlots / 64, 1024><<<groups, 1024, 0, stream>>>(p);
    return hipGetLastError();
  }
  p.count = static_cast<int32_t*>(workspace);
  p.from = p.count + rows;
  p.to = p.from + rows * most;
  if (slots <= 8 * kSelect)
    paged_select_kernel<8, true><<<groups, kSelect, 0, stream>>>(p);
  else if (slots <= 32 * kSelect)
    paged_select_kernel<32, true><<<groups, kSelect, 0, stream>>>(p);
  else
    paged_select_kernel<32, false><<<groups, kSelect, 0, stream>>>(p);
  if (most == 0) return hipGetLastError();
  const int per = kThreads / chunks * 4;
  const unsigned y = static_cast<unsigned>(rows < 65535 ? rows : 65535);
  const dim3 grid(static_cast<unsigned>((most + per - 1) / per), y, static_cast<unsigned>((rows + y - 1) / y));
  paged_move_kernel<<<grid, kThreads, 0, stream>>>(p, per);
  return hipGetLastError();
}

}  // namespace hz
