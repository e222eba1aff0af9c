// Attention of new tokens over paged caches (formulas: include/hz_paged.h; operand layouts: token_device.h).
//
// All rows of query and head that share a key head, up to 32 of them, are the columns of one workgroup's products, and the
// workgroup owns a run of slots, so that a cache is read once. How long a run is, it works out from the rows' real lengths:
// the sum of them over a number of runs that fills the card, so that one long row among short ones is divided as
// finely as many of its length would be coarsely. Its four waves take blocks of 32 slots in turn and
// join their sums in LDS; a row that is one run gets its results there, the others' runs are joined by a second
// kernel. Where the page table leaves no room for long rows, each row is one run and there is no second kernel.
//
// A block is 32 slots on v_mfma_f32_16x16x32_bf16: keys go from memory into the products' registers, values through
// LDS of the wave's own. Where the slots lie is looked up two blocks ahead, so that no load waits for the page table.
//
// Accumulated weights need every row's final maximum and sum: the scores are kept in memory (4 bytes for each row
// and slot beside the 4 D or 8 D that are read) and the second kernel, or the run itself where it is its row, adds up exp2 of them.
#include "paged_launch.h"
#include "token_device.h"

namespace hz {
namespace {

using namespace token;

constexpr int kThreads = 256;
constexpr int kBlock = 32;  // slots of a wave's step
constexpr int kKept = 16;   // slots whose scores are kept row by row

struct PagedParams {
  Pages c;
  hz_token_tensor q;
  void* out;
  const float *slopes, *scores;
  float* scores_out;
  float *partial, *kept;  // workspace: see layout()
  float2 *stats, *norms;  // each run's base and sum; norm_of() of each row
  int B, Nq, H, Hk, G, D, rows, blocks;  // rows: Nq G; blocks of 16 or 32 of them
  int64_t blocks_kept;                   // of a row's kept scores: blocks of kKept slots
  int64_t runs_wanted, runs_fill;        // for one key head and block of rows, over all batch rows: at most, and to fill the card
  const int* plan;                       // of more than 64 batch rows
  int waves, step;                       // waves of a run; slots that they take at a time, of which runs are multiples
  bool whole;                            // each row is one run
  float to_tanh, to_score2, decay;
};

// How the rows are divided: runs of `chunk` slots, at least one a row (more steps than the quotient of all by those wanted, so that the
// further runs are fewer than wanted; longer ones, up to kLong steps, while there are runs enough to fill the card). Run 0 of
// batch row b has number b; the further runs of all rows follow in order. Up to 64 rows, every wave works it out for itself, a length a lane; more rows have it
// worked out once by paged_plan_kernel (512 rows in every wave: 8 us more of a workgroup's time than a lookup).
constexpr int kPlanRows = 64;
struct Found {
  int b, run;
};
__device__ __forceinline__ int further(int n, int chunk) { return n <= chunk ? 0 : (n - 1) / chunk; }
__device__ __forceinline__ int steps_of(const PagedParams& p, int n) { return (n + p.step - 1) / p.step; }
constexpr int kLong = 8;
template <class T>
__device__ __forceinline__ int chunk_of(const PagedParams& p, T steps) {
  T each = steps / static_cast<T>(p.runs_wanted) + 1;
  if (each < kLong) {
    const T fill = steps / static_cast<T>(p.runs_fill) + 1;
    each = fill > kLong ? kLong : fill > each ? fill : each;
  }
  const T most = steps_of(p, p.c.slots);
  return static_cast<int>(each < most ? each : most) * p.step;
}

struct Plan {
  int chunk, all, mine, upto;  // all: number of further runs; this lane's row's, and those of the rows up to it (without a table)
  const int* table;            // chunk, all, [B] the further runs before each row, then their Founds
  __device__ __forceinline__ Plan(const PagedParams& p, int lane) : mine(0), upto(0), table(p.plan) {
    if (p.whole) {
      chunk = p.c.slots;
      all = 0;
      return;
    }
    if (table != nullptr) {
      chunk = table[0];
      all = table[1];
      return;
    }
    const int n = lane < p.B ? p.c.length(lane) : 0;
    // (the steps of 64 rows are below 2^31)
    chunk = chunk_of(p, static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan(steps_of(p, n))), 63)));
    mine = further(n, chunk);
    upto = static_cast<int>(wave_scan(mine));
    all = __builtin_amdgcn_readlane(upto, 63);
  }
  // The batch row of run `at`, and its number there; false behind the last one.
  __device__ __forceinline__ bool find(const PagedParams& p, int at, Found& f) const {
    if (at >= p.B + all) return false;
    if (at < p.B) {
      f = Found{at, 0};
    } else if (table != nullptr) {
      f = reinterpret_cast<const Found*>(table + 2 + (p.B + 1) / 2 * 2)[at - p.B];
    } else {
      const int l = __ffsll(static_cast<unsigned long long>(__ballot(upto > at - p.B))) - 1;
      f = Found{l, 1 + at - p.B - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l))};
    }
    return true;
  }
  // The number of run 1 of batch row b. (Reads other lanes' numbers: all of the wave must be there, also in what encloses the call.)
  __device__ __forceinline__ int second(const PagedParams& p, int b) const {
    return p.B + (table != nullptr ? table[2 + b] : __builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(mine, b));
  }
};

// The table of more than 64 rows. One workgroup.
__global__ void __launch_bounds__(1024) paged_plan_kernel(PagedParams p, int* table) {
  __shared__ int64_t sums[16];
  __shared__ int counts[16];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  int64_t steps = 0;
  for (int b = tid; b < p.B; b += 1024) steps += steps_of(p, p.c.length(b));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) steps += __shfl_xor(steps, d, 64);
  if (lane == 0) sums[wave] = steps;
  __syncthreads();
  steps = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) steps += sums[w];
  const int chunk = chunk_of(p, steps);
  Found* const found = reinterpret_cast<Found*>(table + 2 + (p.B + 1) / 2 * 2);
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 1024) {
    const int b = b0 + tid, more = b < p.B ? further(p.c.length(b), chunk) : 0;
    int x = more;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    if (lane == 63) counts[wave] = x;
    __syncthreads();
    int before = base + x - more;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += counts[w];
      base += counts[w];
    }
    if (b < p.B) table[2 + b] = before;
    for (int r = 0; r < more; ++r) found[before + r] = Found{b, 1 + r};
    __syncthreads();
  }
  if (tid == 0) table[0] = chunk, table[1] = base;
}

// Where a run's results lie: of run number `at`, key head hk and row r of its Nq G.
__device__ __forceinline__ int64_t result_at(const PagedParams& p, int at, int hk, int r) {
  return (static_cast<int64_t>(at) * p.Hk + hk) * p.rows + r;
}

// Where row r's score of a slot is kept: sixteen slots' rows one behind the other, which is what a wave's store writes (a row's
// slots one behind the other: 512 rows of up to 1800 slots 23.3 us to read, 21.0 so; 131072 slots of 24 rows 60.9 us to attend and
// write, 59.5, by 32 slots 60.1).
__device__ __forceinline__ int64_t kept_at(const PagedParams& p, int unit, int r, int slot) {
  return ((unit * p.blocks_kept + slot / kKept) * p.rows + r) * kKept + slot % kKept;
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A step's weights as the products with the values take them. bfloat16: in two parts, 2^-16 off together, so that an output is rounded once. (In one
// part outputs were off by 0.0008 of their size beside that rounding's 0.0017.)
template <int PARTS>
__device__ __forceinline__ auto weight_frag(const v16f& y) {
  if constexpr (PARTS == 1)
    return grad_frag<1>(y, 0);
  else
    return frag_of<3>(y, 0);
}

// A block's values in LDS. bfloat16: a Tile, whose reads transpose. float32: the floats themselves, split into parts as they are read
// (three bfloat16 planes would take half as much again, and a workgroup a CU less); chunk i of four of row r lies at chunk
// i ^ (4 (r / 4 % 2)), so that the rows that a wave reads at once, four apart, lie in both halves of the banks.
template <int DP, int PARTS>
struct Values;
template <int DP>
struct Values<DP, 1> {
  typedef uint16_t Element;
  Element* base;
  __device__ __forceinline__ void put(int row, int chunk, const Raw8<1>& r) const { Tile<kBlock, DP, 1>{base}.put(row, chunk, frag(r)); }
  __device__ __forceinline__ Frag<1> columns(int dt, int lane) const { return Tile<kBlock, DP, 1>{base}.columns16(dt, lane); }
};
template <int DP>
struct Values<DP, 3> {
  typedef float Element;
  Element* base;
  __device__ __forceinline__ static int at(int row, int chunk) { return row * DP + ((chunk ^ ((row >> 2 & 1) << 2)) << 2); }
  __device__ __forceinline__ void put(int row, int chunk, const Raw8<3>& r) const {
    *reinterpret_cast<v4f*>(base + at(row, 2 * chunk)) = r.a;
    *reinterpret_cast<v4f*>(base + at(row, 2 * chunk + 1)) = r.b;
  }
  // Lane 16 g + c gets column 16 dt + c of the rows 16 (j / 4) + 4 g + j % 4.
  __device__ __forceinline__ Frag<3> columns(int dt, int lane) const {
    const int g = lane >> 4, c = lane & 15;
    const float* const from = base + at(4 * g, 4 * dt + (c >> 2)) + (c & 3);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = from[(16 * (j / 4) + j % 4) * DP];
    const Split8 s = split8(x);
    return Frag<3>{{s.h, s.m, s.l}};
  }
};

// Where the 32 slots of a block lie, and the loads of their keys and values into a wave's registers: lane 16 g + c gets of the keys what
// the products' operand wants (rows c and 16 + c, elements 32 s + 8 g .. + 7), and of the values rows lane / CH
// + STEP j. Slots of no page, and behind the run's end, become zeros and are not read.
//
// Keys of bfloat16: a lane's operand is 16 bytes of each 64 of its row, and four lanes reading 64 bytes together make requests of half
// a cache line. Eight lanes read 128 bytes of a row instead, of rows 0 .. 7 and then 8 .. 15, and lanes eight apart
// exchange what belongs to the other (paged_token_long_bf16 260 -> 234 us).
template <int DP, int PARTS>
struct Lanes {
  static constexpr int DS = DP / 32, CH = DP / 8, LOADS = kBlock * CH / 64, STEP = 64 / CH, BYTES = PARTS == 1 ? 2 : 4;
  static constexpr bool TURNED = PARTS == 1 && DS >= 2;
  __device__ __forceinline__ static int key_row(int lane, int s) { return TURNED ? (lane & 7) + 8 * (s & 1) : lane & 15; }
  __device__ __forceinline__ static int key_element(int lane, int s) {
    return TURNED ? 64 * (s / 2) + 8 * (lane >> 4) + (lane & 8 ? 32 : 0) : 32 * s + 8 * (lane >> 4);
  }
  __device__ __forceinline__ static void keys(const Raw8<PARTS> (&raw)[DS], Frag<PARTS> (&k)[DS], int lane) {
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) k[ds] = frag(raw[ds]);
    if constexpr (TURNED) {
      const bool low = (lane & 8) == 0;
#pragma unroll
      for (int ds = 0; ds < DS; ds += 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = k[ds].p[0][i], b = k[ds + 1].p[0][i];
          const uint32_t other = __builtin_amdgcn_mov_dpp(low ? b : a, 0x128, 0xf, 0xf, true);  // of the lane eight on in the sixteen
          k[ds].p[0][i] = low ? a : other;
          k[ds + 1].p[0][i] = low ? other : b;
        }
    }
  }
};

// Pages of a multiple of 16 slots: sixteen slots lie one behind the other. Each half of a block is a buffer whose end the
// hardware checks: base and end are scalars, a lane's offset never changes, and no address is formed in vector registers.
// ONCE: past the caches.
template <int DP, int PARTS, bool APART>
struct Slots : Lanes<DP, PARTS> {
  typedef Lanes<DP, PARTS> L;
  const PagedParams& p;
  const int32_t* table;
  const char *k, *v;  // of the key head
  int stop, lane;
  uint32_t at_k[L::DS], at_v[L::LOADS / 2];
  int page_then[2];  // of the block two on
  struct Half {
    int page, in, count;  // count: its slots
  };
  Half next[2];

  __device__ __forceinline__ Slots(const PagedParams& p_, const int32_t* table_, int hk, int stop_, int lane_, int64_t (*)[kBlock][2])
      : p(p_), table(table_), k(static_cast<const char*>(p_.c.k) + hk * p_.c.head_k * L::BYTES),
        v(static_cast<const char*>(p_.c.v) + hk * p_.c.head_v * L::BYTES), stop(stop_), lane(lane_) {
    constexpr uint32_t kBehind = 0x7fffffffu;  // behind every buffer's end
#pragma unroll
    for (int s = 0; s < L::DS; ++s) {
      const int d = L::key_element(lane, s);
      at_k[s] = d < p.D ? (L::key_row(lane, s) * static_cast<uint32_t>(p.c.token_k) + d) * L::BYTES : kBehind;
    }
#pragma unroll
    for (int j = 0; j < L::LOADS / 2; ++j) {
      const int d = lane % L::CH * 8;
      at_v[j] = d < p.D ? ((lane / L::CH + L::STEP * j) * static_cast<uint32_t>(p.c.token_v) + d) * L::BYTES : kBehind;
    }
  }
  __device__ __forceinline__ void look(int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) page_then[i] = k0 + 16 * i < stop ? table[p.c.page_of(k0 + 16 * i)] : -1;
  }
  // Makes the block looked up the next one; its slots that lie in a page.
  __device__ __forceinline__ uint32_t take(int k0, int) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int slot = k0 + 16 * i, page = __builtin_amdgcn_readfirstlane(page_then[i]);
      next[i].page = page;
      next[i].in = slot - p.c.page_of(slot) * p.c.size;
      next[i].count = page >= 0 && page < p.c.pages ? min(16, stop - slot) : 0;
    }
    return ((1u << next[0].count) - 1) | ((1u << next[1].count) - 1) << 16;
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const char* base, const Half& h, int64_t page, int64_t token) const {
    const int64_t bytes = h.count > 0 ? ((h.count - 1) * token + p.D) * L::BYTES : 0;
    const char* const from = h.count > 0 ? base + (h.page * page + h.in * token) * L::BYTES : base;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(from), 0, static_cast<int>(bytes), 0x00027000);
  }
  template <bool ONCE>
  __device__ __forceinline__ static void one(Raw8<1>& r, __amdgpu_buffer_rsrc_t from, uint32_t at) {
    r.u = __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, ONCE ? 2 : 0);
  }
  template <bool ONCE>
  __device__ __forceinline__ static void one(Raw8<3>& r, __amdgpu_buffer_rsrc_t from, uint32_t at) {
    r.a = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, ONCE ? 2 : 0));
    r.b = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(from, at + 16, 0, ONCE ? 2 : 0));
  }
  template <bool ONCE>
  __device__ __forceinline__ void load_k(Raw8<PARTS> (&rk)[2][L::DS], int) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __amdgpu_buffer_rsrc_t from = buffer(k, next[i], p.c.page_k, p.c.token_k);
#pragma unroll
      for (int s = 0; s < L::DS; ++s) one<ONCE>(rk[i][s], from, at_k[s]);
    }
  }
  template <bool ONCE>
  __device__ __forceinline__ void load_v(Raw8<PARTS> (&rv)[L::LOADS], int) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __amdgpu_buffer_rsrc_t from = buffer(v, next[i], p.c.page_v, p.c.token_v);
#pragma unroll
      for (int j = 0; j < L::LOADS / 2; ++j) one<ONCE>(rv[i * (L::LOADS / 2) + j], from, at_v[j]);
    }
  }
};

// Other pages: every slot is looked up by a lane of its own, and its offsets go to the others through LDS.
template <int DP, int PARTS>
struct Slots<DP, PARTS, true> : Lanes<DP, PARTS> {
  typedef Lanes<DP, PARTS> L;
  const PagedParams& p;
  const int32_t* table;
  int hk, stop, lane, page_then;
  int64_t (*where)[kBlock][2];  // two blocks' offsets of keys and values; -1: no page

  __device__ __forceinline__ Slots(const PagedParams& p_, const int32_t* table_, int hk_, int stop_, int lane_, int64_t (*where_)[kBlock][2])
      : p(p_), table(table_), hk(hk_), stop(stop_), lane(lane_), where(where_) {}
  __device__ __forceinline__ void look(int k0) {
    const int slot = k0 + (lane & 31);
    page_then = slot < stop ? table[p.c.page_of(slot)] : -1;
  }
  __device__ __forceinline__ uint32_t take(int k0, int buffer) {
    const int slot = k0 + (lane & 31), in = slot - p.c.page_of(slot) * p.c.size;
    const bool known = page_then >= 0 && page_then < p.c.pages;
    if (lane < 32) {
      where[buffer][lane][0] = known ? page_then * p.c.page_k + in * p.c.token_k : -1;
      where[buffer][lane][1] = known ? page_then * p.c.page_v + in * p.c.token_v : -1;
    }
    wave_fence();
    return static_cast<uint32_t>(__ballot(known));
  }
  template <bool ONCE>
  __device__ __forceinline__ static void one(Raw8<PARTS>& r, const void* base, int64_t at, bool on) {
    if constexpr (ONCE)
      r.u = on ? __builtin_nontemporal_load(reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(base) + at)) : v4u{0u, 0u, 0u, 0u};
    else
      r.load(base, at, on);
  }
  template <bool ONCE>
  __device__ __forceinline__ void load_k(Raw8<PARTS> (&rk)[2][L::DS], int buffer) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int s = 0; s < L::DS; ++s) {
        const int64_t at = where[buffer][16 * i + L::key_row(lane, s)][0];
        const int d = L::key_element(lane, s);
        one<ONCE>(rk[i][s], p.c.k, at + hk * p.c.head_k + d, at >= 0 && d < p.D);
      }
  }
  template <bool ONCE>
  __device__ __forceinline__ void load_v(Raw8<PARTS> (&rv)[L::LOADS], int buffer) const {
#pragma unroll
    for (int j = 0; j < L::LOADS; ++j) {
      const int64_t at = where[buffer][lane / L::CH + L::STEP * j][1];
      const int d = lane % L::CH * 8;
      one<ONCE>(rv[j], p.c.v, at + hk * p.c.head_v + d, at >= 0 && d < p.D);
    }
  }
};
// A run of slots and who has it. waves 4: the workgroup; waves 1: each wave one of its own, and they share nothing.
struct Run {
  bool together, alone;  // alone: its row has no other
  int wave, id, b, hk, r0, n, begin, first, stop;
  const int32_t* table;
  // Of blocks of `rows` rows of query and head. False behind the last run.
  __device__ __forceinline__ bool find(const PagedParams& p, const Plan& plan, int wave_, int rows) {
    wave = __builtin_amdgcn_readfirstlane(wave_);
    together = p.waves > 1;
    id = together ? static_cast<int>(blockIdx.x) : 4 * static_cast<int>(blockIdx.x) + wave;
    hk = id % p.Hk;
    id /= p.Hk;
    r0 = id % p.blocks * rows;
    id /= p.blocks;
    Found found;
    if (!plan.find(p, id, found)) return false;
    b = found.b;
    n = p.c.length(b);
    alone = n <= plan.chunk;
    begin = found.run * plan.chunk;
    stop = alone ? n : min(n, begin + plan.chunk);
    first = begin + (together ? kBlock * wave : 0);
    table = p.c.table + static_cast<int64_t>(b) * p.c.width;
    return true;
  }
  // Whether most of its pages (64 of them, evenly spread, where there are more) lie at the same place of the row before or behind, whose workgroups
  // then read them too. Rows that share pages without being neighbours are not seen.
  __device__ __forceinline__ bool shares(const PagedParams& p, int lane) const {
    if (begin >= stop) return false;
    const int page0 = p.c.page_of(begin), count = p.c.page_of(stop - 1) - page0 + 1, some = min(count, 64);
    const int32_t* const at = table + page0 + static_cast<int64_t>(min(lane, some - 1)) * count / some;
    const int own = *at, before = b > 0 ? *(at - p.c.width) : -1, behind = b + 1 < p.B ? *(at + p.c.width) : -1;
    const uint64_t votes = __ballot(lane < some && own >= 0 && own < p.c.pages && (own == before || own == behind));
    return 2 * static_cast<int>(__popcll(votes)) > some;
  }
};

// Where chunk ch of four outputs of column x lies among sixteen columns: the columns' writes go to different banks.
template <int DP>
__device__ __forceinline__ int out_at(int x, int ch) { return x * DP + (ch ^ (x & 7)) * 4; }

// What a row's weights are formed by: its largest score and one over its sum of exp2(score - largest). Apart: one number for both, the largest plus
// the sum's logarithm, would be rounded at the size of the score, an error of 2^-24 of it in all weights of the row. (A row that sees no
// slot has weights 0, one with a NaN has NaN.)
__device__ __forceinline__ float2 norm_of(float top, float sum) { return make_float2(top == kNegInf ? 0.f : top, sum == 0.f ? 0.f : 1.f / sum); }

// The results of a run: rows r0 .. r0 + columns - 1 from its waves' sums of values (out_at, o_wave floats a wave) and their base and sum
// (sums_wave pairs a wave). Where the run is its row and weights are added up, what they are formed by goes to norms and to
// memory.
template <int DP, int PARTS>
__device__ __forceinline__ void put_run(const PagedParams& p, const Run& run, const float* o, int o_wave, const float2* sums, int sums_wave, int columns, int r0,
                                        float2* norms) {
  const int w0 = run.together ? 0 : run.wave, threads = 64 * p.waves;
  for (int x = run.together ? threadIdx.x : threadIdx.x & 63; x < columns * (DP / 4); x += threads) {
    const int col = x / (DP / 4), ch = x % (DP / 4), r = r0 + col, d = 4 * ch;
    if (d >= p.D) continue;
    float top = kNegInf, all = 0.f;
    for (int w = w0; w < w0 + p.waves; ++w) top = fmaxf(top, sums[w * sums_wave + col].x);
    const float base = top == kNegInf ? 0.f : top;
    v4f y = zero4();
    for (int w = w0; w < w0 + p.waves; ++w) {
      const float2 s = sums[w * sums_wave + col];
      const float a = fast_exp2(s.x - base);
      all += a * s.y;
      y += a * *reinterpret_cast<const v4f*>(o + w * o_wave + out_at<DP>(col, ch));
    }
    if (run.alone) {
      const int64_t at = (static_cast<int64_t>(run.b) * p.Nq + r / p.G) * p.H + run.hk * p.G + r % p.G;
      const float inv = all > 0.f || all != all ? 1.f / all : 0.f;
      store_four<PARTS>(p.out, at * p.D + d, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
      if (p.kept != nullptr && ch == 0) {
        norms[col] = norm_of(top, all);
        if (p.norms != nullptr) p.norms[at] = norms[col];
      }
    } else {
      const int64_t to = result_at(p, run.id, run.hk, r);
      *reinterpret_cast<v4f*>(p.partial + to * p.D + d) = y;
      if (ch == 0) p.stats[to] = make_float2(top, all);
    }
  }
}

// The weights of four slots of a row of n, from what rows r0 .. r0 + rows - 1 of query and head kept.
__device__ __forceinline__ void add_kept(const PagedParams& p, int unit, int slot, const float2* norms, int r0, int rows, v4f& sum) {
  const float* const kept = p.kept + kept_at(p, unit, r0, slot);
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    const v4f x = *reinterpret_cast<const v4f*>(kept + r * kKept);
    const float2 norm = norms[r];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = fmaf(fast_exp2(x[e] - norm.x), norm.y, sum[e]);
  }
}
__device__ __forceinline__ void put_weights(const PagedParams& p, int unit, int n, int slot, const v4f& sum) {
  const int64_t at = static_cast<int64_t>(unit) * p.c.slots + slot;
  if (slot + 4 <= p.c.slots && p.c.slots % 4 == 0) {
    v4f x = zero4();
    if (slot < n && p.scores != nullptr) x = p.decay * *reinterpret_cast<const v4f*>(p.scores + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = slot + e < n ? x[e] + sum[e] : 0.f;
    *reinterpret_cast<v4f*>(p.scores_out + at) = x;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (slot + e >= p.c.slots) break;
    float x = 0.f;
    if (slot + e < n) x = sum[e] + (p.scores != nullptr ? p.decay * p.scores[at + e] : 0.f);
    p.scores_out[at + e] = x;
  }
}

// The weights of a run that is its row, and all rows of query and head, by its threads.
__device__ __forceinline__ void put_own_weights(const PagedParams& p, const Run& run, const float2* norms) {
  run.together ? __syncthreads() : wave_fence();
  const int threads = 64 * p.waves, unit = run.b * p.Hk + run.hk;
  for (int slot = 4 * (run.together ? threadIdx.x : threadIdx.x & 63); slot < p.c.slots; slot += 4 * threads) {
    v4f sum = zero4();
    if (slot < run.n) add_kept(p, unit, slot, norms, 0, p.rows, sum);
    put_weights(p, unit, run.n, slot, sum);
  }
}

// Of the lane some places on in the row of sixteen.
template <int CONTROL>
__device__ __forceinline__ float row_turned(float x) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), CONTROL, 0xf, 0xf, true));
}

// Which reads go past the caches. float32 none (16 x 8192 slots of 8 heads of 128: 203 us, 214 past them), nor bfloat16 where several workgroups read
// a run (more than 32 rows of query and head). Else bfloat16 does (16 rows of up to 32768 slots of 8 heads of 128: 241 us, 267 through
// them; in pages of 100 slots 241 and 268, of one slot 253 and 279), but for runs whose pages the rows beside read too (16 x 32768 slots: 346 us;
// four fifths of the pages shared 283 past the caches, 230 as asked of each run; all of them 268, 181). Rows that are one run each are not asked,
// which takes 1 us (64 x 900 slots 46.7, 47.7; all of them shared 27.1 past the caches, 27.3 through them; 1024 x 1000 apart 635, 704).
enum Past { kNone, kUnshared, kAll };

template <int DP, int PARTS, bool CAP, int CB, bool APART, Past PAST>
__global__ void __launch_bounds__(kThreads, PARTS == 1 ? 2 : 1) paged_attention_kernel(PagedParams p) {
  typedef Slots<DP, PARTS, APART> S;
  constexpr int DS = S::DS, DT = DP / 16, CH = S::CH, LOADS = S::LOADS, STEP = S::STEP;
  typedef Values<DP, PARTS> V;
  __shared__ __align__(16) typename V::Element v_lds[4][kBlock * DP];
  __shared__ __align__(16) int64_t where_lds[APART ? 4 : 1][2][kBlock][2];
  __shared__ float2 sums_lds[4][16 * CB];  // each wave's base and sum
  __shared__ float2 norms_lds[4][16 * CB];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const V vt{v_lds[wave]};
  const Plan plan(p, lane);
  Run run;
  if (!run.find(p, plan, wave, 16 * CB)) return;  // all waves of the run
  const bool together = run.together;
  const int b = run.b, n = run.n, hk = run.hk, r0 = run.r0, first = run.first, stop = run.stop, step = p.step;
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
  float m[CB], l[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = kNegInf, l[cb] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[cb][dt] = zero4();
  }

  S slots(p, run.table, hk, stop, lane, where_lds[APART ? wave : 0]);
  if (first < stop) slots.look(first);
  auto attend = [&](auto once) __attribute__((always_inline)) {
    const int lr = lane / CH, lc = lane % CH;
    Raw8<PARTS> rk[2][DS], rv[LOADS];
    uint32_t known = 0, known_next = 0;  // slots of the block at hand, and of the next, that lie in a page
    int buffer = 0;
    if (first < stop) {
      known = slots.take(first, 0);
      slots.look(first + step);
      slots.template load_v<once.value>(rv, 0);
      slots.template load_k<once.value>(rk, 0);
      known_next = slots.take(first + step, 1);
    }
    for (int k0 = first; k0 < stop; k0 += step, buffer ^= 1) {
      const bool more = k0 + step < stop;
      slots.look(k0 + 2 * step);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) vt.put(lr + STEP * j, lc, rv[j]);
      if (more) slots.template load_v<once.value>(rv, buffer ^ 1);
      v4f s[CB][2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        Frag<PARTS> k[DS];
        S::keys(rk[kb], k, lane);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          s[cb][kb] = zero4();
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) s[cb][kb] = mma16(k[ds], q[cb][ds], s[cb][kb]);
        }
      }
      if (more) slots.template load_k<once.value>(rk, buffer ^ 1);
      settle(s);
      wave_fence();
      const uint32_t known_then = slots.take(k0 + 2 * step, buffer);  // what this block needed of it has been read
      Frag<PARTS == 1 ? 2 : 3> w[CB];
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
          float* const to = p.kept + kept_at(p, b * p.Hk + hk, row[cb], k1);
          *reinterpret_cast<v4f*>(to) = v4f{x[0], x[1], x[2], x[3]};
          *reinterpret_cast<v4f*>(to + kKept * p.rows) = v4f{x[4], x[5], x[6], x[7]};
        }
        top = group_max(top);
        if (__any(top > m[cb])) {
          const float now = fmaxf(m[cb], top), alpha = m[cb] == kNegInf ? 0.f : fast_exp2(m[cb] - now);
          m[cb] = now;
          l[cb] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[cb][dt] *= alpha;
        }
        const float base = m[cb] == kNegInf ? 0.f : m[cb];
        v16f y = v16f{};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = fast_exp2(x[i] - base);
          l[cb] += y[i];
        }
        w[cb] = weight_frag<PARTS>(y);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const Frag<PARTS> v = vt.columns(dt, lane);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) o[cb][dt] = mma16(v, w[cb], o[cb][dt]);
      }
      wave_fence();
      known = known_next;
      known_next = known_then;
    }
  };
  if constexpr (PAST == kUnshared)
    run.shares(p, lane) ? attend(std::false_type{}) : attend(std::true_type{});
  else
    attend(std::bool_constant<PAST == kAll>{});
  settle(o);
  // the run's sums, sixteen columns at a time, through the values' LDS
  float* const mine = reinterpret_cast<float*>(v_lds[wave]);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float sum = group_sum(l[cb]);
    if (g == 0) sums_lds[wave][16 * cb + c] = make_float2(m[cb], sum);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<v4f*>(mine + out_at<DP>(c, 4 * dt + g)) = o[cb][dt];
    together ? __syncthreads() : wave_fence();
    put_run<DP, PARTS>(p, run, reinterpret_cast<const float*>(v_lds[0]), kBlock * DP * static_cast<int>(sizeof(typename V::Element)) / 4,
                       sums_lds[0] + 16 * cb, 16 * CB, min(16, p.rows - r0 - 16 * cb), r0 + 16 * cb, norms_lds[together ? 0 : wave] + 16 * cb);
    if (cb + 1 < CB) together ? __syncthreads() : wave_fence();
  }
  if (p.kept != nullptr && p.norms == nullptr) put_own_weights(p, run, norms_lds[together ? 0 : wave]);
}

// The same for float32 and one or two rows of query and head, on vector instructions: a lane has a part of each key's dot product, as
// its loads bring it, and of the values' sums over its slots; the weights go from the one to the other through LDS. The matrix cores
// would take sixteen rows for one or two and have keys and values split into three parts each: 512 rows of up to 225 slots of 8 heads
// of 64 took 59 us so with one row, 63 with two and 68 on the matrix cores; 16 of up to 8192 of 8 heads of 128 took 122, 125 and 147.
// Four rows took 94 (matrix cores 68) and 144 (148). Heads of 32: 28, 30 and 38. bfloat16 gains nothing (31.0 us with one row of 64,
// 32.6 on the matrix cores; 120 and 120 with heads of 128). Heads of 64 keep two workgroups a CU (three spill: 73 us); heads of 128
// need the registers of one.
template <int DP, bool CAP, int R, bool APART>
__global__ void __launch_bounds__(kThreads, DP <= 64 ? 2 : 1) paged_rows_kernel(PagedParams p) {
  typedef Slots<DP, 3, APART> S;
  constexpr int DS = S::DS, CH = S::CH, LOADS = S::LOADS, STEP = S::STEP;
  __shared__ __align__(16) int64_t where_lds[APART ? 4 : 1][2][kBlock][2];
  __shared__ __align__(16) float w_lds[4][R][kBlock], o_lds[4][R * DP];
  __shared__ float2 sums_lds[4][R];
  __shared__ float2 norms_lds[4][R];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const Plan plan(p, lane);
  Run run;
  if (!run.find(p, plan, wave, R)) return;  // all waves of the run
  const int b = run.b, n = run.n, stop = run.stop, step = p.step, hk = run.hk;
  float q[R][DS][8], slope2[R];
  int pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = r / p.G, h = hk * p.G + r % p.G;
    pos[r] = n - p.Nq + i;
    slope2[r] = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      Raw8<3> x;
      const int d = S::key_element(lane, s);
      x.load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + d, d < p.D);
      floats(x, q[r][s]);
    }
  }
  float o[R][8] = {}, m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) m[r] = kNegInf, l[r] = 0.f;
  S slots(p, run.table, hk, stop, lane, where_lds[APART ? wave : 0]);
  const int lr = lane / CH, lc = lane % CH;
  Raw8<3> rk[2][DS], rv[LOADS];
  uint32_t known = 0, known_next = 0;
  int buffer = 0;
  if (run.first < stop) {
    slots.look(run.first);
    known = slots.take(run.first, 0);
    slots.look(run.first + step);
    slots.template load_k<false>(rk, 0);
    slots.template load_v<false>(rv, 0);
    known_next = slots.take(run.first + step, 1);
  }
  for (int k0 = run.first; k0 < stop; k0 += step, buffer ^= 1) {
    const bool more = k0 + step < stop;
    slots.look(k0 + 2 * step);
    float x[R][2] = {};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        float k[8];
        floats(rk[kb][s], k);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[r][kb] = fmaf(k[e], q[r][s][e], x[r][kb]);
      }
    if (more) slots.template load_k<false>(rk, buffer ^ 1);
    const uint32_t seen = known;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = kNegInf;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int at = 16 * kb + c, key = k0 + at;
        float y = xor32_pair_sum(xor16_pair_sum(x[r][kb]));
        y = CAP ? tanh_of<3>(y * p.to_tanh) * p.to_score2 : y * p.to_score2;
        if (slope2[r] != 0.f) y -= slope2[r] * static_cast<float>(abs(pos[r] - key));
        y = key <= pos[r] && (seen >> at & 1) ? y : kNegInf;
        x[r][kb] = y;
        top = fmaxf(top, y);
        if (p.kept != nullptr && g == 0)
          p.kept[kept_at(p, b * p.Hk + hk, r, key)] = y;
      }
      if (__any(top > m[r])) {
        top = fmaxf(top, row_turned<0x121>(top));
        top = fmaxf(top, row_turned<0x122>(top));
        top = fmaxf(top, row_turned<0x124>(top));
        top = fmaxf(top, row_turned<0x128>(top));
        const float now = fmaxf(m[r], top), alpha = m[r] == kNegInf ? 0.f : fast_exp2(m[r] - now);
        m[r] = now;
        l[r] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[r][e] *= alpha;
      }
      const float base = m[r] == kNegInf ? 0.f : m[r];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float w = fast_exp2(x[r][kb] - base);
        l[r] += w;
        if (g == 0) w_lds[wave][r][16 * kb + c] = w;
      }
    }
    wave_fence();
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      float v[8];
      floats(rv[j], v);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = w_lds[wave][r][lr + STEP * j];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
      }
    }
    if (more) slots.template load_v<false>(rv, buffer ^ 1);
    wave_fence();
    known = known_next;
    known_next = slots.take(k0 + 2 * step, buffer);  // (the next block's loads are under way)
  }
  // a row's sum over the sixteen lanes that have different slots; the values' over the lanes that have the same elements
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float sum = l[r];
    sum += row_turned<0x128>(sum);
    sum += row_turned<0x124>(sum);
    sum += row_turned<0x122>(sum);
    sum += row_turned<0x121>(sum);
    if (lane == 0) sums_lds[wave][r] = make_float2(m[r], sum);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y = o[r][e];
      if constexpr (CH <= 8) y += row_turned<0x128>(y);
      if constexpr (CH <= 4) y += row_turned<0x124>(y);
      o[r][e] = xor32_pair_sum(xor16_pair_sum(y));
    }
    if (lane < CH) {
      *reinterpret_cast<v4f*>(o_lds[wave] + out_at<DP>(r, 2 * lc)) = v4f{o[r][0], o[r][1], o[r][2], o[r][3]};
      *reinterpret_cast<v4f*>(o_lds[wave] + out_at<DP>(r, 2 * lc + 1)) = v4f{o[r][4], o[r][5], o[r][6], o[r][7]};
    }
  }
  run.together ? __syncthreads() : wave_fence();
  put_run<DP, 3>(p, run, o_lds[0], R * DP, sums_lds[0], R, p.rows, 0, norms_lds[run.together ? 0 : wave]);
  if (p.kept != nullptr && p.norms == nullptr) put_own_weights(p, run, norms_lds[run.together ? 0 : wave]);
}

// The run results of one row of (b, i, h).
struct Runs {
  int64_t first, others;  // where the first run's lie, and behind it those of run 1 on, `step` apart
  int64_t step;
  int count;
  __device__ __forceinline__ Runs(const PagedParams& p, int count_, int second, int b, int hk, int r)
      : first(result_at(p, b, hk, r)), others(result_at(p, second - 1, hk, r)), step(static_cast<int64_t>(p.Hk) * p.rows), count(count_) {}
  __device__ __forceinline__ int64_t at(int run) const { return run == 0 ? first : others + run * step; }
};

// Behind the attention, in one launch. Workgroups 0 .. joins - 1 join the runs of rows that have several: 4 * lanes elements of a row of
// (b, i, h) at a time, 256 / lanes ways taking the runs in turn. lanes 8, four workgroups to a row of 128
// elements, where there are few rows (115 runs of 96 rows 6.6 us, 12 with a workgroup a row); else 32 (12 runs of 512 rows 5.7 us,
// 9 with four). The others add up the weights that each slot has had, 1024 slots of a row and key head a workgroup,
// four a thread.
constexpr int kRowTile = 64;
template <int PARTS>
__global__ void __launch_bounds__(kThreads) paged_finish_kernel(PagedParams p, int joins, int lanes, int per_row) {
  __shared__ __align__(16) float o_lds[4][32][4];
  __shared__ float m_lds[4], l_lds[4];
  __shared__ float2 norms_lds[kRowTile];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const Plan plan(p, lane);
  if (static_cast<int>(blockIdx.x) < joins) {
    if (plan.all == 0) return;
    const int way = tid / lanes, ways = kThreads / lanes, dl = tid % lanes;
    const int per = p.Nq * p.H, quarters = (p.D + 4 * lanes - 1) / (4 * lanes);
    for (int64_t unit = blockIdx.x; unit < static_cast<int64_t>(p.B) * per * quarters; unit += joins) {
      const int64_t at = unit / quarters;
      const int d = (static_cast<int>(unit % quarters) * lanes + dl) * 4, b = static_cast<int>(at / per), n = p.c.length(b);
      if (n <= plan.chunk) continue;  // all of the workgroup
      const int within = static_cast<int>(at - static_cast<int64_t>(b) * per), i = within / p.H, h = within % p.H;
      const Runs runs(p, 1 + further(n, plan.chunk), plan.second(p, b), b, h / p.G, i * p.G + h % p.G);
      float m = kNegInf, l = 0.f;
      v4f o = zero4();
      for (int r = way; r < runs.count; r += 4 * ways) {  // four loads under way
        float2 st[4];
        v4f y[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int64_t from = runs.at(min(r + x * ways, runs.count - 1));
          st[x] = p.stats[from];
          y[x] = *reinterpret_cast<const v4f*>(p.partial + from * p.D + (d < p.D ? d : 0));
        }
        float now = m;
#pragma unroll
        for (int x = 0; x < 4; ++x) now = fmaxf(now, st[x].x);
        const float base = now == kNegInf ? 0.f : now, alpha = fast_exp2(m - base);
        m = now, l *= alpha, o *= alpha;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (r + x * ways >= runs.count) break;
          const float a = fast_exp2(st[x].x - base);  // (a weight of zero passes a NaN on too)
          l += a * st[x].y;
          o += a * y[x];
        }
      }
      float now = m;
      for (int x = lanes; x < 64; x <<= 1) now = fmaxf(now, __shfl_xor(now, x, 64));
      const float alpha = fast_exp2(m - (now == kNegInf ? 0.f : now));
      l *= alpha, o *= alpha;
      for (int x = lanes; x < 64; x <<= 1) {
        l += __shfl_xor(l, x, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x, 64);
      }
      if (lane < lanes) *reinterpret_cast<v4f*>(o_lds[wave][dl]) = o;
      if (lane == 0) m_lds[wave] = now, l_lds[wave] = l;
      __syncthreads();
      if (tid < lanes) {
        const float top = fmaxf(fmaxf(m_lds[0], m_lds[1]), fmaxf(m_lds[2], m_lds[3])), base = top == kNegInf ? 0.f : top;
        o = zero4(), l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float a = fast_exp2(m_lds[w] - base);
          o += a * *reinterpret_cast<const v4f*>(o_lds[w][dl]);
          l += a * l_lds[w];
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        if (d < p.D) store_four<PARTS>(p.out, at * p.D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      }
      __syncthreads();
    }
    return;
  }
  const int id = static_cast<int>(blockIdx.x) - joins, unit = id / per_row;
  const int b = unit / p.Hk, hk = unit % p.Hk, n = p.c.length(b);
  const int slot0 = id % per_row * (4 * kThreads), slot = slot0 + 4 * tid;
  const int count = 1 + further(n, plan.chunk), second = count > 1 ? plan.second(p, b) : 0;  // (before lanes go different ways)
  v4f sum = zero4();
  for (int r0 = 0; r0 < p.rows && slot0 < n; r0 += kRowTile) {
    const int rows = min(kRowTile, p.rows - r0);
    if (r0 > 0) __syncthreads();
    // what each row's weights are formed by: eight lanes a row
    const int d8 = tid & 7;
    for (int r = tid >> 3; r < rows; r += kThreads / 8) {
      const int i = (r0 + r) / p.G, g = (r0 + r) % p.G;
      float2 norm;
      if (count == 1) {
        norm = p.norms[(static_cast<int64_t>(b) * p.Nq + i) * p.H + hk * p.G + g];
      } else {
        const Runs runs(p, count, second, b, hk, r0 + r);
        float m = kNegInf, l = 0.f;
        for (int x0 = d8; x0 < runs.count; x0 += 64) {  // eight loads under way
          float2 st[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) st[x] = p.stats[runs.at(min(x0 + 8 * x, runs.count - 1))];
          float now = m;
#pragma unroll
          for (int x = 0; x < 8; ++x) now = fmaxf(now, st[x].x);
          const float base = now == kNegInf ? 0.f : now;
          l *= fast_exp2(m - base);
#pragma unroll
          for (int x = 0; x < 8; ++x) l += x0 + 8 * x < runs.count ? fast_exp2(st[x].x - base) * st[x].y : 0.f;
          m = now;
        }
        float now = m;
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) now = fmaxf(now, __shfl_xor(now, x, 64));
        l *= fast_exp2(m - (now == kNegInf ? 0.f : now));
        m = now;
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) l += __shfl_xor(l, x, 64);
        norm = norm_of(m, l);
      }
      if (d8 == 0) norms_lds[r] = norm;
    }
    __syncthreads();
    if (slot < n) add_kept(p, unit, slot, norms_lds, r0, rows, sum);
  }
  if (slot < p.c.slots) put_weights(p, unit, n, slot, sum);
}

// Workgroups that fill the card: the rows are divided so that there are about kFill, three for each place of most kernels (half as many
// take 16% longer where rows are long, paged_token_long_bf16; twice as many 3%). While a workgroup's run is below kLong steps
// they are as few as kLeast (16 x 8192 float32 slots of 8 heads of 128: 150 us, 178 by kFill alone).
// Where there are rows of key heads for all its waves, kAlone, each wave has one to itself and shares nothing
// (512 rows of up to 225 float32 slots of 8 heads of 64: 75 -> 62 us).
// Rows of at most kWhole slots, by the width of their page table, or twice as many where there is a workgroup for each of the card's
// units, are not divided: no table of runs, and no second kernel, as a run adds up its own weights (512 rows of up to 225 slots of 8
// float32 heads of 64: 48 us, 60 with three kernels; 64 of 900 of bfloat16: 20, 25; 32 of 1000: 20, 27). Below a workgroup a unit, 4
// rows of 450 take 8.9 us, or 9.9 in two kernels, and a launch less; of 777 11.7, or 10.0; 20 of 1000 of bfloat16 16.9, or 14.0. float32 on
// the matrix cores takes twice the time a slot (4 rows of 500 of heads of 128: 22, or 15), so half as many.
constexpr int64_t kFill = 1536, kLeast = 512, kAlone = 2048, kWhole = 512, kUnits = 256;

struct Layout {
  int64_t rows, block, blocks, waves, step, runs_wanted, runs_fill, runs, blocks_kept, partial, stats, kept, norms, plan, total;
  bool whole, table, finish_weights;  // each row is one run; a table of the runs; weights by the second kernel
};

// Rows of query and head in a workgroup's products: 16, or 32 where there are more; float32 heads of more than 64 elements have
// no registers for 32, and read their keys and values again for every 16.
// The workspace, in floats: partial outputs and statistics of every run, kept scores, what each row's weights are formed by.
Layout layout(const hz_paged_attention_args& a) {
  const hz_paged_cache& c = a.cache;
  Layout w{};
  const int64_t slots = c.page_size * c.table_width;
  w.rows = a.Nq * (a.H / c.Hk);
  w.block = w.rows <= 16 || (c.dtype == HZ_DTYPE_F32 && c.D > 64) ? 16 : 32;
  w.blocks = (w.rows + w.block - 1) / w.block;
  const int64_t units = c.B * c.Hk * w.blocks;
  w.waves = units >= kAlone ? 1 : 4;
  w.step = w.waves * kBlock;
  const int64_t wanted = (w.waves == 1 ? kAlone : kFill) / (c.Hk * w.blocks), longest = (slots + w.step - 1) / w.step;
  w.runs_wanted = wanted > 1 ? wanted : 1;
  const int64_t fill = (w.waves == 1 ? kAlone : kLeast) / (c.Hk * w.blocks);
  w.runs_fill = fill > 1 ? fill : 1;
  // runs are at least (all lengths) / wanted and step long: each row has one, and all together less than `wanted` more
  const int64_t most = c.B * longest;
  const bool in_parts = c.dtype == HZ_DTYPE_F32 && w.rows > 2;  // float32 on the matrix cores
  w.whole = slots <= (units >= kUnits ? 2 * kWhole : in_parts ? kWhole / 2 : kWhole);
  w.runs = w.whole ? c.B : w.runs_wanted + c.B < most ? w.runs_wanted + c.B : most;
  auto take = [&](int64_t floats) {
    const int64_t at = w.total;
    w.total += (floats + 3) / 4 * 4;
    return at;
  };
  w.partial = take(w.whole ? 0 : w.runs * c.Hk * w.rows * c.D);
  w.stats = take(w.whole ? 0 : w.runs * c.Hk * w.rows * 2);
  w.table = !w.whole && c.B > kPlanRows;
  w.plan = take(w.table ? 2 + (c.B + 1) / 2 * 2 + 2 * (w.runs - c.B) : 0);
  w.blocks_kept = (slots + kBlock - 1) / kBlock * (kBlock / kKept);
  if (a.scores_out != nullptr) {
    w.kept = take(c.B * c.Hk * w.rows * w.blocks_kept * kKept);
    w.finish_weights = !w.whole || w.blocks > 1;
    w.norms = take(w.finish_weights ? 2 * c.B * a.Nq * a.H : 0);
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
  PagedParams p{Pages(c), a.q, a.out, a.slopes, a.scores, a.scores_out, ws + w.partial, want ? ws + w.kept : nullptr,
                reinterpret_cast<float2*>(ws + w.stats), w.finish_weights ? reinterpret_cast<float2*>(ws + w.norms) : nullptr,
                static_cast<int>(c.B), static_cast<int>(a.Nq),
                static_cast<int>(a.H), static_cast<int>(c.Hk), static_cast<int>(a.H / c.Hk), static_cast<int>(c.D),
                static_cast<int>(w.rows), static_cast<int>(w.blocks), w.blocks_kept, w.runs_wanted, w.runs_fill,
                w.table ? reinterpret_cast<int*>(ws + w.plan) : nullptr, static_cast<int>(w.waves), static_cast<int>(w.step), w.whole,
                capped ? a.scale / a.softcap : 0.f, (capped ? a.softcap : a.scale) * kLog2e, a.decay};
  const unsigned grid = static_cast<unsigned>(w.waves > 1 ? w.runs * c.Hk * w.blocks : (w.runs * c.Hk * w.blocks + 3) / 4);
  if (w.table) paged_plan_kernel<<<1, 1024, 0, stream>>>(p, reinterpret_cast<int*>(ws + w.plan));
  // sixteen slots as a buffer: one behind the other, apart, within 31 bits
  const int64_t least = c.k.token < c.v.token ? c.k.token : c.v.token, most = c.k.token > c.v.token ? c.k.token : c.v.token;
  const bool buffers = c.page_size % 16 == 0 && least >= c.D && most < int64_t(1) << 24;
  auto attend = [&](auto apart) {
    constexpr bool APART = apart.value;
    if constexpr (PARTS == 3)
      if (w.rows <= 2) {
        if (w.rows == 1)
          paged_rows_kernel<DP, CAP, 1, APART><<<grid, kThreads, 0, stream>>>(p);
        else
          paged_rows_kernel<DP, CAP, 2, APART><<<grid, kThreads, 0, stream>>>(p);
        return;
      }
    auto attend16 = [&](auto past) { paged_attention_kernel<DP, PARTS, CAP, 1, APART, past.value><<<grid, kThreads, 0, stream>>>(p); };
    auto attend32 = [&](auto past) { paged_attention_kernel<DP, PARTS, CAP, 2, APART, past.value><<<grid, kThreads, 0, stream>>>(p); };
    typedef std::integral_constant<Past, kNone> None;
    typedef std::integral_constant<Past, kUnshared> Unshared;
    typedef std::integral_constant<Past, kAll> All;
    if constexpr (PARTS == 3) {
      if (w.block == 16)
        attend16(None{});
      else if constexpr (DP < 128)
        attend32(None{});
    } else if (w.block == 16) {  // (up to 16 rows are one block)
      w.whole ? attend16(All{}) : attend16(Unshared{});
    } else if (w.blocks == 1) {
      w.whole ? attend32(All{}) : attend32(Unshared{});
    } else {
      attend32(None{});
    }
  };
  buffers ? attend(std::false_type{}) : attend(std::true_type{});
  const int64_t outputs = !w.whole && w.runs > c.B ? c.B * a.Nq * a.H : 0;  // where a row may have several runs
  const int lanes = outputs * ((c.D + 31) / 32) <= 1024 ? 8 : 32;
  const int64_t units = lanes == 8 ? outputs * ((c.D + 31) / 32) : outputs;
  const int joins = static_cast<int>(units < 2048 ? units : 2048), per_row = (p.c.slots + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t finish = joins + (w.finish_weights ? c.B * c.Hk * per_row : 0);
  if (finish > 0) paged_finish_kernel<PARTS><<<static_cast<unsigned>(finish), kThreads, 0, stream>>>(p, joins, lanes, per_row);
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
