// Paged caches: new tokens into their slots, and eviction by accumulated weight (include/hz_paged.h).
//
// Append: a thread copies 16 bytes of a key or value; bound by those bytes.
//
// Eviction, of each row and key head: (1) one workgroup finds the budget's smallest weight by its bits, eight at a time
// from the top, with a histogram in LDS for each; (2) each wave goes over its own stretch of the
// slots: it counts, and after one exchange of the counts it knows the number of each of its holes and
// late survivors without further waiting; (3) a second kernel moves the survivors behind the budget into the holes
// below it. Sources lie behind the budget and targets below it, so the moves do not depend on each other, and what
// stays below is not touched: about budget (1 - budget / n) tokens are read and written and not the whole
// budget, which a compaction in order would move.
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

constexpr int kSelect = 1024;  // threads of a row's workgroup
constexpr int kWaves = kSelect / 64;

struct EvictParams {
  Pages c;
  const float* scores;
  float* scores_out;
  int32_t *sources, *lengths_out;
  int32_t *count, *from, *to;  // of each row and key head: its moves
  int B, Hk, budget, keep, sinks, recent, most;  // keep: min(budget, slots); most: moves at most
};

// The order of scores as unsigned numbers; NaN is the least, -0 equals 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

// Exclusive sum over the workgroup's waves of one number a wave; total: over all.
__device__ __forceinline__ int before_wave(int mine, int* lds, int& total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  __syncthreads();
  if (lane == 0) lds[wave] = mine;
  __syncthreads();
  int sum = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) sum += lds[w];
    total += lds[w];
  }
  return sum;
}

__global__ void __launch_bounds__(kSelect) paged_select_kernel(EvictParams p) {
  __shared__ int hist[256], shared[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / p.Hk);
  const int n = p.c.length(b), m = p.budget, slots = p.c.slots;
  const float* const scores = p.scores + row * slots;
  float* const scores_out = p.scores_out + row * slots;
  int32_t* const sources = p.sources + row * p.keep;
  if (tid == 0 && row % p.Hk == 0) p.lengths_out[b] = min(n, m);
  for (int s = min(n, m) + tid; s < slots; s += kSelect) {
    scores_out[s] = 0.f;
    if (s < p.keep) sources[s] = -1;
  }
  if (n <= m) {
    for (int s = tid; s < n; s += kSelect) scores_out[s] = scores[s], sources[s] = s;
    if (tid == 0) p.count[row] = 0;
    return;
  }
  // the threshold: of the slots lo .. hi - 1 those above it stay, and the first `equal` of those at it
  const int lo = p.sinks, hi = n - p.recent, need = m - p.sinks - p.recent;
  uint32_t threshold = 0;
  int equal = need;  // still wanted among the scores whose top bits are the threshold's
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int s = lo + tid; s < hi; s += kSelect) {
        const uint32_t u = ordered(scores[s]);
        if (shift == 24 || (u ^ threshold) >> (shift + 8) == 0) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      // sums from the top bin down; each thread of the first four waves has one bin
      int above = 0;
      if (tid < 256) {
        const int bin = 255 - tid;
        int x = hist[bin];
        const int mine = x;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int y = __shfl_up(x, d, 64);
          if (lane >= d) x += y;
        }
        above = x - mine;
        if (lane == 63) shared[wave] = x;
      }
      __syncthreads();
      if (tid < 256) {
        for (int w = 0; w < wave; ++w) above += shared[w];
        const int mine = hist[255 - tid];
        if (above < equal && above + mine >= equal) shared[4] = 255 - tid, shared[5] = above;
      }
      __syncthreads();
      threshold |= static_cast<uint32_t>(shared[4]) << shift;
      equal -= shared[5];
      __syncthreads();
    }
  }
  // each wave's stretch of the slots
  const int each = ((n + kWaves - 1) / kWaves + 63) / 64 * 64, first = min(n, wave * each), last = min(n, first + each);
  auto is_equal = [&](int s, uint32_t u) { return need > 0 && s >= lo && s < hi && u == threshold; };
  auto is_kept = [&](int s, uint32_t u) { return s < lo || s >= hi || (need > 0 && u > threshold); };
  int total, equals = 0;
  for (int s = first + lane; s - lane < last; s += 64)
    equals += __popcll(__ballot(s < last && is_equal(s, ordered(scores[s < last ? s : 0]))));
  const int equal_before = before_wave(equals, shared, total);
  const uint64_t below = (uint64_t(1) << lane) - 1;
  // what each wave has of holes and of late survivors, then their places in the lists
  auto pass = [&](auto take) {
    int eq = equal_before;
    for (int s = first + lane; s - lane < last; s += 64) {
      const bool in = s < last;
      const float x = scores[in ? s : 0];
      const uint32_t u = ordered(x);
      const bool at = in && is_equal(s, u);
      const uint64_t votes = __ballot(at);
      const bool stays = in && (is_kept(s, u) || (at && eq + __popcll(votes & below) < equal));
      eq += __popcll(votes);
      take(s, x, stays, __ballot(in && s < m && !stays), __ballot(stays && s >= m));
    }
  };
  int holes = 0, lates = 0;
  pass([&](int, float, bool, uint64_t hole, uint64_t late) { holes += __popcll(hole), lates += __popcll(late); });
  holes = before_wave(holes, shared, total);
  const int late_before = before_wave(lates, shared, total);
  lates = late_before;
  int32_t* const from = p.from + row * p.most;
  int32_t* const to = p.to + row * p.most;
  pass([&](int s, float x, bool stays, uint64_t hole, uint64_t late) {
    if (hole >> lane & 1) to[holes + __popcll(hole & below)] = s;
    if (late >> lane & 1) from[lates + __popcll(late & below)] = s;
    if (stays && s < m) sources[s] = s, scores_out[s] = x;
    holes += __popcll(hole);
    lates += __popcll(late);
  });
  __syncthreads();
  for (int i = tid; i < total; i += kSelect) {
    const int s = to[i], at = from[i];
    sources[s] = at;
    scores_out[s] = scores[at];
  }
  if (tid == 0) p.count[row] = total;
}

// Moves of one row and key head: `chunks` lanes of 16 bytes a key and a value.
__global__ void __launch_bounds__(kThreads) paged_move_kernel(EvictParams p, int chunks, int bytes, int per_block) {
  const int64_t row = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
  if (row >= static_cast<int64_t>(p.B) * p.Hk) return;
  const int count = p.count[row], b = static_cast<int>(row / p.Hk), h = static_cast<int>(row % p.Hk);
  const int begin = blockIdx.x * per_block, end = min(count, begin + per_block);
  const int32_t* const table = p.c.table + static_cast<int64_t>(b) * p.c.width;
  const int rows = kThreads / chunks, ch = threadIdx.x % chunks;
  if (static_cast<int>(threadIdx.x) >= rows * chunks) return;
  for (int i = begin + static_cast<int>(threadIdx.x) / chunks; i < end; i += rows) {
    const int at = p.from[row * p.most + i], to = p.to[row * p.most + i];
    const int pa = p.c.page_of(at), pt = p.c.page_of(to);
    const int page_a = table[pa], page_t = table[pt];
    if (page_a < 0 || page_a >= p.c.pages || page_t < 0 || page_t >= p.c.pages) continue;
    const int in_a = at - pa * p.c.size, in_t = to - pt * p.c.size;
    char* const k = static_cast<char*>(const_cast<void*>(p.c.k)) + 16 * ch;
    char* const v = static_cast<char*>(const_cast<void*>(p.c.v)) + 16 * ch;
    const uint4 x = *reinterpret_cast<const uint4*>(k + (page_a * p.c.page_k + in_a * p.c.token_k + h * p.c.head_k) * bytes);
    const uint4 y = *reinterpret_cast<const uint4*>(v + (page_a * p.c.page_v + in_a * p.c.token_v + h * p.c.head_v) * bytes);
    *reinterpret_cast<uint4*>(k + (page_t * p.c.page_k + in_t * p.c.token_k + h * p.c.head_k) * bytes) = x;
    *reinterpret_cast<uint4*>(v + (page_t * p.c.page_v + in_t * p.c.token_v + h * p.c.head_v) * bytes) = y;
  }
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
  return a.cache.B * a.cache.Hk * (1 + 2 * most_moves(a)) * static_cast<int64_t>(sizeof(int32_t));
}

hipError_t launch_paged_evict(const hz_paged_evict_args& a, void* workspace, hipStream_t stream) {
  const hz_paged_cache& c = a.cache;
  const int64_t rows = c.B * c.Hk, most = most_moves(a), slots = c.page_size * c.table_width;
  EvictParams p{Pages(c), a.scores, a.scores_out, a.sources, a.lengths_out, nullptr, nullptr, nullptr,
                static_cast<int>(c.B), static_cast<int>(c.Hk), static_cast<int>(a.budget),
                static_cast<int>(a.budget < slots ? a.budget : slots), static_cast<int>(a.sinks),
                static_cast<int>(a.recent), static_cast<int>(most)};
  p.count = static_cast<int32_t*>(workspace);
  p.from = p.count + rows;
  p.to = p.from + rows * most;
  paged_select_kernel<<<static_cast<unsigned>(rows), kSelect, 0, stream>>>(p);
  if (most == 0) return hipGetLastError();
  const int bytes = bytes_of(c.dtype), chunks = static_cast<int>(c.D) * bytes / 16, per = kThreads / chunks * 8;
  const unsigned y = static_cast<unsigned>(rows < 65535 ? rows : 65535);
  const dim3 grid(static_cast<unsigned>((most + per - 1) / per), y, static_cast<unsigned>((rows + y - 1) / y));
  paged_move_kernel<<<grid, kThreads, 0, stream>>>(p, chunks, bytes, per);
  return hipGetLastError();
}

}  // namespace hz
