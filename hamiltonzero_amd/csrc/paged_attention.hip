// Attention of new tokens over paged caches (formulas: include/hz_paged.h; operand layouts: token_device.h).
//
// All rows of query and head that share a key head, up to 32 of them, are the columns of one wave's products, and a wave
// owns a run of slots, so that a cache is read once. How long a run is, each wave works out from the rows' real lengths:
// the sum of them over a number of runs that fills the card, so that one long row among
// short ones is divided as finely as many of its length would be coarsely. A row that is one run gets its results at once; the
// others' runs are joined by a second kernel.
//
// 32 slots at a time on v_mfma_f32_16x16x32_bf16: keys go from memory into the products' registers, values through
// LDS of the wave's own. Where the slots lie is looked up two blocks ahead, so that no load waits for the page table.
//
// Accumulated weights need every row's final maximum and sum: the scores are kept in memory (4 bytes for each row
// and slot beside the 4 D or 8 D that are read) and a third kernel adds up exp2 of them.
#include "paged_launch.h"
#include "token_device.h"

namespace hz {
namespace {

using namespace token;

constexpr int kThreads = 256;
constexpr int kBlock = 32;  // slots of a wave's step

struct PagedParams {
  Pages c;
  hz_token_tensor q;
  void* out;
  const float *slopes, *scores;
  float* scores_out;
  float *partial, *stats, *kept, *lse;  // workspace: see layout()
  int B, Nq, H, Hk, G, D, rows, blocks;  // rows: Nq G; blocks of 32 of them
  int64_t slots_kept;                    // of a row of kept scores: the slots, rounded up to 32
  int64_t runs_wanted;                   // for one key head and block of rows, over all batch rows
  float cap, to_tanh, to_score2, decay;
};

// How the rows are divided: runs of `chunk` slots; those of batch row b are the numbers first .. first + runs - 1.
struct Plan {
  int chunk;
  __device__ __forceinline__ static int runs(int n, int chunk) { return n <= chunk ? 1 : (n + chunk - 1) / chunk; }
  __device__ __forceinline__ Plan(const PagedParams& p, int lane) {
    int64_t sum = 0;
    for (int b = lane; b < p.B; b += 64) sum += p.c.length(b);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
    const int64_t each = (sum + p.runs_wanted - 1) / p.runs_wanted;
    chunk = static_cast<int>(each < 1 ? kBlock : (each + kBlock - 1) / kBlock * kBlock);
  }
  // The batch row of run `at`, and its number there; false behind the last one.
  __device__ __forceinline__ bool find(const PagedParams& p, int64_t at, int lane, int& b, int& run) const {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int mine = b0 + lane < p.B ? runs(p.c.length(b0 + lane), chunk) : 0;
      int x = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
      }
      const uint64_t behind = __ballot(base + x > at);
      if (behind != 0) {
        const int l = __ffsll(static_cast<unsigned long long>(behind)) - 1;
        b = b0 + l;
        run = static_cast<int>(at - base) - (__builtin_amdgcn_readlane(x, l) - __builtin_amdgcn_readlane(mine, l));
        return true;
      }
      base += __builtin_amdgcn_readlane(x, 63);
    }
    return false;
  }
  // The first run of batch row b.
  __device__ __forceinline__ int64_t first(const PagedParams& p, int b, int lane) const {
    int64_t sum = 0;
    for (int x = lane; x < b; x += 64) sum += runs(p.c.length(x), chunk);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
    return sum;
  }
};

// Where a run's results lie: of batch-wide run number `at`, key head hk and row r of its Nq G.
__device__ __forceinline__ int64_t result_at(const PagedParams& p, int64_t at, int hk, int r) {
  return (at * p.Hk + hk) * p.rows + r;
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int DP, int PARTS, bool CAP, int CB>
__global__ void __launch_bounds__(kThreads, PARTS == 1 ? 2 : 1) paged_attention_kernel(PagedParams p) {
  constexpr int DS = DP / 32, DT = DP / 16, CH = DP / 8, LOADS = kBlock * CH / 64, STEP = 64 / CH;
  typedef Tile<kBlock, DP, PARTS> V;
  __shared__ __align__(16) uint16_t v_lds[4][V::kPlane * PARTS];
  __shared__ __align__(16) int64_t where_lds[4][2][kBlock][2];  // offsets of a block's keys and values; -1: no page
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const V vt{v_lds[wave]};
  int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int hk = static_cast<int>(id % p.Hk);
  id /= p.Hk;
  const int r0 = static_cast<int>(id % p.blocks) * 32;
  id /= p.blocks;
  const Plan plan(p, lane);
  int b, run_id;
  if (!plan.find(p, id, lane, b, run_id)) return;  // waves share nothing: no barriers
  const int n = p.c.length(b);
  const bool alone = n <= plan.chunk;
  const int first = run_id * plan.chunk, stop = alone ? n : min(n, first + plan.chunk);
  const int32_t* const table = p.c.table + static_cast<int64_t>(b) * p.c.width;

  Frag<PARTS> q[CB][DS];
  int pos[CB], row[CB];
  float slope2[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    row[cb] = min(r0 + 16 * cb + c, p.rows - 1);
    const int i = row[cb] / p.G, h = hk * p.G + row[cb] % p.G;
    pos[cb] = n - p.Nq + i;
    slope2[cb] = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      Raw8<PARTS> r;
      const int d = 32 * s + 8 * g;
      r.load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + d, d < p.D);
      q[cb][s] = frag(r);
    }
  }
  v4f o[CB][DT];
  float m[CB], l[CB], l_exact[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = kNegInf, l[cb] = l_exact[cb] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[cb][dt] = zero4();
  }

  // slots k0 .. k0 + 31: lanes 0 .. 31 look up a slot each
  auto page_at = [&](int k0) {
    const int slot = k0 + (lane & 31);
    return slot < stop ? table[p.c.page_of(slot)] : -1;
  };
  auto put_where = [&](int k0, int page) -> uint32_t {
    const int slot = k0 + (lane & 31), in = slot - p.c.page_of(slot) * p.c.size;
    const bool known = page >= 0 && page < p.c.pages;
    if (lane < 32) {
      where_lds[wave][(k0 >> 5) & 1][lane][0] = known ? page * p.c.page_k + in * p.c.token_k : -1;
      where_lds[wave][(k0 >> 5) & 1][lane][1] = known ? page * p.c.page_v + in * p.c.token_v : -1;
    }
    return static_cast<uint32_t>(__ballot(known));
  };
  const int lr = lane / CH, lc = lane % CH;
  Raw8<PARTS> rk[2][DS], rv[LOADS];
  auto load_k = [&](int k0) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int64_t at = where_lds[wave][(k0 >> 5) & 1][16 * kb + c][0];
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const int d = 32 * s + 8 * g;
        rk[kb][s].load(p.c.k, at + hk * p.c.head_k + d, at >= 0 && d < p.D);
      }
    }
  };
  auto load_v = [&](int k0) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int64_t at = where_lds[wave][(k0 >> 5) & 1][lr + STEP * j][1];
      rv[j].load(p.c.v, at + hk * p.c.head_v + 8 * lc, at >= 0 && 8 * lc < p.D);
    }
  };
  uint32_t known = 0, known_next = 0;  // slots of the block at hand, and of the next, that lie in a page
  if (first < stop) {
    known = put_where(first, page_at(first));
    known_next = put_where(first + 32, page_at(first + 32));
    wave_fence();
    load_v(first);
    load_k(first);
  }
  for (int k0 = first; k0 < stop; k0 += 32) {
    const int page_next = page_at(k0 + 64);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) vt.put(lr + STEP * j, lc, frag(rv[j]));
    if (k0 + 32 < stop) load_v(k0 + 32);
    v4f s[CB][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      Frag<PARTS> k[DS];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) k[ds] = frag(rk[kb][ds]);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        s[cb][kb] = zero4();
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) s[cb][kb] = mma16(k[ds], q[cb][ds], s[cb][kb]);
      }
    }
    if (k0 + 32 < stop) load_k(k0 + 32);
    settle(s);
    wave_fence();
    const uint32_t known_then = put_where(k0 + 64, page_next);  // this block's offsets have all been read
    Frag<PARTS> w[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const int k1 = k0 + 4 * g;
      float x[8], top = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 16 * (i / 4) + i % 4, key = k1 + at;
        x[i] = s[cb][i / 4][i % 4];
        x[i] = CAP ? tanh_of<PARTS>(x[i] * p.to_tanh) * p.to_score2 : x[i] * p.to_score2;
        if (slope2[cb] != 0.f) x[i] -= slope2[cb] * static_cast<float>(abs(pos[cb] - key));
        x[i] = key <= pos[cb] && (known >> (at + 4 * g) & 1) ? x[i] : kNegInf;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
      if (p.kept != nullptr && r0 + 16 * cb + c < p.rows) {
        float* const to = p.kept + (static_cast<int64_t>(b * p.Hk + hk) * p.rows + row[cb]) * p.slots_kept + k1;
        *reinterpret_cast<v4f*>(to) = v4f{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<v4f*>(to + 16) = v4f{x[4], x[5], x[6], x[7]};
      }
      top = group_max(top);
      if (__any(top > m[cb])) {
        const float now = fmaxf(m[cb], top), alpha = m[cb] == kNegInf ? 0.f : fast_exp2(m[cb] - now);
        m[cb] = now;
        l[cb] *= alpha;
        l_exact[cb] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[cb][dt] *= alpha;
      }
      const float base = m[cb] == kNegInf ? 0.f : m[cb];
      v16f y = v16f{};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = fast_exp2(x[i] - base);
        l_exact[cb] += y[i];
      }
      w[cb] = frag_of<PARTS>(y, 0);
      add_weights(w[cb], y, 0, l[cb]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const Frag<PARTS> v = vt.columns16(dt, lane);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o[cb][dt] = mma16(v, w[cb], o[cb][dt]);
    }
    wave_fence();
    known = known_next;
    known_next = known_then;
  }
  settle(o);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float sum = group_sum(l[cb]), exact = group_sum(l_exact[cb]);
    if (r0 + 16 * cb + c >= p.rows) continue;
    if (alone) {
      const int i = row[cb] / p.G, h = hk * p.G + row[cb] % p.G;
      const int64_t at = (static_cast<int64_t>(b) * p.Nq + i) * p.H + h;
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int d = 16 * dt + 4 * g;
        if (d < p.D) store_four<PARTS>(p.out, at * p.D + d, o[cb][dt][0] * inv, o[cb][dt][1] * inv, o[cb][dt][2] * inv, o[cb][dt][3] * inv);
      }
      if (p.kept != nullptr && g == 0) p.lse[at] = exact > 0.f ? m[cb] + log2f(exact) : 0.f;
      continue;
    }
    const int64_t to = result_at(p, id, hk, row[cb]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * dt + 4 * g;
      if (d < p.D) *reinterpret_cast<v4f*>(p.partial + to * p.D + d) = o[cb][dt];
    }
    if (g == 0) *reinterpret_cast<v4f*>(p.stats + to * 4) = v4f{m[cb], sum, exact, 0.f};
  }
}

// Joins the runs of rows that have several: eight half waves a row of (b, i, h), four elements a lane.
template <int PARTS>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(PagedParams p) {
  constexpr int WAYS = 8;
  __shared__ __align__(16) float o_lds[WAYS][HZ_TOKEN_MAX_HEAD];
  __shared__ float l_lds[WAYS][2];
  const int lane = threadIdx.x & 31, way = threadIdx.x >> 5, d = 4 * lane;
  const Plan plan(p, threadIdx.x & 63);
  const int64_t at = blockIdx.x;
  const int b = static_cast<int>(at / (static_cast<int64_t>(p.Nq) * p.H)), n = p.c.length(b);
  if (n <= plan.chunk) return;
  const int64_t first = plan.first(p, b, threadIdx.x & 63);
  const int runs = Plan::runs(n, plan.chunk);
  const int within = static_cast<int>(at - static_cast<int64_t>(b) * p.Nq * p.H), i = within / p.H, h = within % p.H, hk = h / p.G;
  const int64_t from = result_at(p, first, hk, i * p.G + h % p.G), step = static_cast<int64_t>(p.Hk) * p.rows;
  float m = kNegInf, l = 0.f, exact = 0.f;
  v4f o = zero4();
#pragma unroll 4
  for (int r = lane; r < runs; r += 32) m = fmaxf(m, p.stats[(from + r * step) * 4]);
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const float base = m == kNegInf ? 0.f : m;
#pragma unroll 4
  for (int r = way; r < runs; r += WAYS) {
    const v4f st = *reinterpret_cast<const v4f*>(p.stats + (from + r * step) * 4);
    const float a = fast_exp2(st[0] - base);
    l += a * st[1];
    exact += a * st[2];
    if (d < p.D) o += a * *reinterpret_cast<const v4f*>(p.partial + (from + r * step) * p.D + d);
  }
  *reinterpret_cast<v4f*>(&o_lds[way][d]) = o;
  if (lane == 0) l_lds[way][0] = l, l_lds[way][1] = exact;
  __syncthreads();
  if (way != 0) return;
#pragma unroll
  for (int x = 1; x < WAYS; ++x) {
    l += l_lds[x][0];
    exact += l_lds[x][1];
    o += *reinterpret_cast<const v4f*>(&o_lds[x][d]);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  if (d < p.D) store_four<PARTS>(p.out, at * p.D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (p.kept != nullptr && lane == 0) p.lse[at] = exact > 0.f ? m + log2f(exact) : 0.f;
}

// The weights that each slot has had: 1024 slots of a row and key head a workgroup, four a thread.
__global__ void __launch_bounds__(kThreads) paged_weights_kernel(PagedParams p, int per_row) {
  const int64_t unit = blockIdx.x / per_row;
  const int b = static_cast<int>(unit / p.Hk), hk = static_cast<int>(unit % p.Hk);
  const int slot = (static_cast<int>(blockIdx.x) % per_row * kThreads + static_cast<int>(threadIdx.x)) * 4, n = p.c.length(b);
  if (slot >= p.c.slots) return;
  v4f sum = zero4();
  if (slot < n) {
    const float* const kept = p.kept + unit * p.rows * p.slots_kept + slot;
#pragma unroll 4
    for (int r = 0; r < p.rows; ++r) {
      const float lse = p.lse[(static_cast<int64_t>(b) * p.Nq + r / p.G) * p.H + hk * p.G + r % p.G];
      const v4f x = *reinterpret_cast<const v4f*>(kept + r * p.slots_kept);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += fast_exp2(x[e] - lse);
    }
  }
  const int64_t at = unit * p.c.slots + slot;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (slot + e >= p.c.slots) break;
    float x = 0.f;
    if (slot + e < n) x = sum[e] + (p.scores != nullptr ? p.decay * p.scores[at + e] : 0.f);
    p.scores_out[at + e] = x;
  }
}

// Waves that fill the card: a row of one key head is divided so that there are about as many.
constexpr int64_t kWaves = 6144;

struct Layout {
  int64_t rows, blocks, runs_wanted, runs, slots_kept, partial, stats, kept, lse, total;
};

// The workspace, in floats: partial outputs and statistics of every run, kept scores, a base and sum for each row.
Layout layout(const hz_paged_attention_args& a) {
  const hz_paged_cache& c = a.cache;
  Layout w{};
  const int64_t slots = c.page_size * c.table_width;
  w.rows = a.Nq * (a.H / c.Hk);
  w.blocks = (w.rows + 31) / 32;
  const int64_t wanted = kWaves / (c.Hk * w.blocks), longest = (slots + kBlock - 1) / kBlock;
  w.runs_wanted = wanted > 1 ? wanted : 1;
  // runs are at least (all lengths) / wanted long, and at least one block: each row has one, and all together at most `wanted` more
  const int64_t most = c.B * longest;
  w.runs = w.runs_wanted + c.B < most ? w.runs_wanted + c.B : most;
  auto take = [&](int64_t floats) {
    const int64_t at = w.total;
    w.total += (floats + 3) / 4 * 4;
    return at;
  };
  w.partial = take(w.runs * c.Hk * w.rows * c.D);
  w.stats = take(w.runs * c.Hk * w.rows * 4);
  w.slots_kept = longest * kBlock;
  if (a.scores_out != nullptr) {
    w.kept = take(c.B * c.Hk * w.rows * w.slots_kept);
    w.lse = take(c.B * a.Nq * a.H);
  }
  return w;
}

template <int DP, int PARTS, bool CAP>
hipError_t run(const hz_paged_attention_args& a, void* workspace, hipStream_t stream) {
  const hz_paged_cache& c = a.cache;
  const Layout w = layout(a);
  float* const ws = static_cast<float*>(workspace);
  const bool want = a.scores_out != nullptr;
  const bool capped = a.softcap > 0.f;
  PagedParams p{Pages(c), a.q, a.out, a.slopes, a.scores, a.scores_out, ws + w.partial, ws + w.stats,
                want ? ws + w.kept : nullptr, want ? ws + w.lse : nullptr, static_cast<int>(c.B), static_cast<int>(a.Nq),
                static_cast<int>(a.H), static_cast<int>(c.Hk), static_cast<int>(a.H / c.Hk), static_cast<int>(c.D),
                static_cast<int>(w.rows), static_cast<int>(w.blocks), w.slots_kept, w.runs_wanted, a.softcap,
                capped ? a.scale / a.softcap : 0.f, (capped ? a.softcap : a.scale) * kLog2e, a.decay};
  const unsigned grid = static_cast<unsigned>((w.runs * c.Hk * w.blocks + 3) / 4);
  if (w.rows <= 16)
    paged_attention_kernel<DP, PARTS, CAP, 1><<<grid, kThreads, 0, stream>>>(p);
  else
    paged_attention_kernel<DP, PARTS, CAP, 2><<<grid, kThreads, 0, stream>>>(p);
  if (w.slots_kept > kBlock) paged_join_kernel<PARTS><<<static_cast<unsigned>(c.B * a.Nq * a.H), kThreads, 0, stream>>>(p);
  if (want) {
    const int per_row = static_cast<int>((p.c.slots + 4 * kThreads - 1) / (4 * kThreads));
    paged_weights_kernel<<<static_cast<unsigned>(c.B * c.Hk * per_row), kThreads, 0, stream>>>(p, per_row);
  }
  return hipGetLastError();
}

}  // namespace

int64_t paged_attention_workspace(const hz_paged_attention_args& a) { return layout(a).total * static_cast<int64_t>(sizeof(float)); }

hipError_t launch_paged_attention(const hz_paged_attention_args& a, void* workspace, hipStream_t stream) {
  auto by_type = [&](auto dp) {
    constexpr int DP = dp.value;
    if (a.cache.dtype == HZ_DTYPE_BF16)
      return a.softcap > 0.f ? run<DP, 1, true>(a, workspace, stream) : run<DP, 1, false>(a, workspace, stream);
    return a.softcap > 0.f ? run<DP, 3, true>(a, workspace, stream) : run<DP, 3, false>(a, workspace, stream);
  };
  if (a.cache.D <= 32) return by_type(std::integral_constant<int, 32>{});
  if (a.cache.D <= 64) return by_type(std::integral_constant<int, 64>{});
  return by_type(std::integral_constant<int, 128>{});
}

}  // namespace hz
