// Forward of the token attention (formulas and masks: include/hz_token.h; operand layouts:
// token_device.h).
//
// Many queries: a workgroup of four waves owns 128 queries of a head, 32 a wave, and streams the keys they
// can see through LDS in tiles of KB with the running maximum and sum of the softmax. bfloat16 tiles
// are copied straight into one of two LDS buffers while the other is used; float32 ones pass through
// registers, where they are split. Tiles that no query of the workgroup can see (behind the last visible key,
// or of other documents) are not visited; a wave forms masks only in tiles where some pair is hidden. Where
// there are few workgroups and many keys, the keys are divided and the parts joined by a second kernel. Bound by the
// exponentials' and the cap's vector work beside the products: attn_prompt_bf16 (2 x 4096 tokens, 16 on 4 heads of 128,
// causal, capped) 196 us, 700 TFLOP/s; 173 without the cap's tanh, 168 without either of the products.
//
// Few queries (at most 32 rows of query and head share a key head): a wave owns a run of keys and
// all of those rows, so the cache is read once, and the same second kernel joins the runs. Bound by those bytes:
// attn_token_long_bf16 (16 rows of 32768 keys, 8 key heads of 128) 265 us, 4.9 to 5.1 TB/s.
#include "token_device.h"

namespace hz {
namespace token {

// One wave a tile of 64 keys.
__global__ void __launch_bounds__(256) doc_tiles_kernel(Params p, DocTile* tiles, int per_row) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int b = static_cast<int>(id / per_row);
  if (b >= p.B) return;
  const int t = static_cast<int>(id - static_cast<int64_t>(b) * per_row), key = t * kDocTile + lane;
  const int doc = key < kv_length(p, b) ? key_document(p, b, key) : -1;
  int lo, hi;
  document_range(doc, lo, hi);
  const bool pad = __any(doc < 0);
  if (lane == 0) tiles[id] = DocTile{lo, hi, pad, 0};
}

// How long a block of queries (the first B nq waves) or keys takes, roughly: the tiles of 64 keys, or of queries by
// position, that hold one of its documents, as one of 256 bins, the longest in bin 0. One wave a block.
__global__ void __launch_bounds__(256) block_bins_kernel(Params p, const DocTile* tiles, int per_row, int nq, int nk, int* bins) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6), queries = static_cast<int64_t>(p.B) * nq;
  if (id >= queries + static_cast<int64_t>(p.B) * nk) return;
  const int lane = threadIdx.x & 63;
  const bool keys = id >= queries;
  const int64_t e = keys ? id - queries : id;
  const int blocks = keys ? nk : nq, b = static_cast<int>(e / blocks);
  const int n = kv_length(p, b);
  const int first = static_cast<int>(e - static_cast<int64_t>(b) * blocks) * kOrderBlock + (keys ? 0 : n - p.Nq);
  const int last = min(first + kOrderBlock, n) - 1;
  const DocTile* const row = tiles + static_cast<int64_t>(b) * per_row;
  int lo = 2147483647, hi = -1, count = 0;
  for (int t = max(first, 0) / kDocTile; t <= (last >= 0 ? last / kDocTile : -1); ++t) {
    const DocTile d = row[t];
    lo = min(lo, d.lo);
    hi = max(hi, d.hi);
  }
  const int from = keys && p.causal ? first / kDocTile : 0, to = !keys && p.causal ? last / kDocTile : per_row - 1;
  if (hi >= 0)
    for (int t = from; t <= to; t += 64) {
      DocTile d{2147483647, -1, 0, 0};
      if (t + lane <= to) d = row[t + lane];
      count += __popcll(__ballot(d.lo <= hi && d.hi >= lo));
    }
  if (lane == 0) bins[id] = 255 - min(255, static_cast<int>(256LL * count / (per_row + 1)));
}

// The blocks' numbers by their bins: workgroup 0 the queries', workgroup 1 the keys'. Which of a bin's blocks comes first is left
// open: it changes when a block's work begins, and nothing of it.
__global__ void __launch_bounds__(1024) block_order_kernel(const int* bins, int* order, int64_t queries, int64_t keys) {
  __shared__ int place[256];
  const int tid = threadIdx.x;
  const int64_t first = blockIdx.x == 0 ? 0 : queries, n = blockIdx.x == 0 ? queries : keys;
  if (tid < 256) place[tid] = 0;
  __syncthreads();
  for (int64_t i = tid; i < n; i += 1024) atomicAdd(&place[bins[first + i] & 255], 1);
  __syncthreads();
  if (tid < 64) {
    int c[4], sum = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) c[x] = place[4 * tid + x], sum += c[x];
    int before = sum;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
      const int y = __shfl_up(before, x, 64);
      if (tid >= x) before += y;
    }
    before -= sum;
#pragma unroll
    for (int x = 0; x < 4; ++x) place[4 * tid + x] = before, before += c[x];
  }
  __syncthreads();
  for (int64_t i = tid; i < n; i += 1024) order[first + atomicAdd(&place[bins[first + i] & 255], 1)] = static_cast<int>(i);
}

static int64_t doc_tiles_per_row(int64_t Nk) { return (Nk + kDocTile - 1) / kDocTile; }

// Documents of different lengths make blocks of different lengths, and a long one that begins late keeps the others
// waiting: taken longest first, where the workgroups do not all run at once (two a CU). attn_train_packed_bf16's forward
// 172 us -> 152, with its gradients 815 -> 741; the two kernels that make the order take 4 us each.
static bool ordered(const hz_token_attention& a) {
  return a.documents != nullptr && a.B * a.H * ((a.Nq + kOrderBlock - 1) / kOrderBlock) > 512;
}

int64_t doc_bytes(const hz_token_attention& a) {
  if (a.documents == nullptr) return 0;
  const int64_t blocks = a.B * ((a.Nq + kOrderBlock - 1) / kOrderBlock + (a.Nk + kOrderBlock - 1) / kOrderBlock);
  return a.B * doc_tiles_per_row(a.Nk) * static_cast<int64_t>(sizeof(DocTile)) + (ordered(a) ? 2 * blocks * static_cast<int64_t>(sizeof(int)) : 0);
}

hipError_t launch_docs(const hz_token_attention& a, Params& p, bool keys, void* memory, hipStream_t stream) {
  if (a.documents == nullptr) return hipSuccess;
  const int64_t per_row = doc_tiles_per_row(a.Nk), n = a.B * per_row;
  DocTile* const tiles = static_cast<DocTile*>(memory);
  doc_tiles_kernel<<<static_cast<unsigned>((n + 3) / 4), 256, 0, stream>>>(p, tiles, static_cast<int>(per_row));
  if (!ordered(a)) return hipGetLastError();
  const int nq = static_cast<int>((a.Nq + kOrderBlock - 1) / kOrderBlock);
  const int nk = keys ? static_cast<int>((a.Nk + kOrderBlock - 1) / kOrderBlock) : 0;
  const int64_t blocks = a.B * (nq + nk);
  int* const bins = reinterpret_cast<int*>(tiles + n);
  int* const order = bins + blocks;
  block_bins_kernel<<<static_cast<unsigned>((blocks + 3) / 4), 256, 0, stream>>>(p, tiles, static_cast<int>(per_row), nq, nk, bins);
  block_order_kernel<<<keys ? 2 : 1, 1024, 0, stream>>>(bins, order, a.B * nq, a.B * nk);
  p.q_order = order;
  p.k_order = keys ? order + a.B * nq : nullptr;
  return hipGetLastError();
}

}  // namespace token
namespace {

using namespace token;

constexpr int kThreads = 256;
constexpr int kQB = kOrderBlock;  // queries a workgroup

// Keys a tile: three parts of 64 keys at 128 elements would leave room for one workgroup a CU.
template <int DP, int PARTS>
constexpr int kKeys = (DP == 128 && PARTS == 3) ? 32 : 64;

// One lane's running softmax of one query, base 2.
struct Running {
  float m = kNegInf, l = 0.f;
};

// A score is a base-2 number s, or, where there is a cap and no distance bias, u = 1 / (1 + e^2y) with
// s = cap2 - 2 cap2 u (tanh y = 1 - 2 u), so that the map to the exponent of 2 is one fused operation.
// Hidden pairs are -inf, or u = +inf.
template <int PARTS, bool CAP, bool SLOPE, bool U, int N>
__device__ __forceinline__ void scores(v16f (&s)[N], const Params& p, const Sight& me, float slope2, int k0, int hh,
                                       bool masked, const int* docs) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (U)
        s[n][i] = __builtin_amdgcn_rcpf(1.f + fast_exp2(s[n][i] * p.to_exp2));
      else if constexpr (CAP)
        s[n][i] = tanh_of<PARTS>(s[n][i] * p.to_tanh) * p.to_score2;
      else
        s[n][i] *= p.to_score2;
    }
  if constexpr (SLOPE) {
    const float at = static_cast<float>(me.pos - k0 - 4 * hh);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] -= slope2 * fabsf(at - static_cast<float>(32 * n + row_of(i, 0)));
  }
  constexpr float kHidden = U ? -kNegInf : kNegInf;
  if (masked) {
    const int last = me.last - k0 - 4 * hh;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] = 32 * n + row_of(i, 0) <= last ? s[n][i] : kHidden;
    if (docs != nullptr) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 d = *reinterpret_cast<const int4*>(docs + 32 * n + 8 * g + 4 * hh);
          s[n][4 * g] = d.x == me.doc ? s[n][4 * g] : kHidden;
          s[n][4 * g + 1] = d.y == me.doc ? s[n][4 * g + 1] : kHidden;
          s[n][4 * g + 2] = d.z == me.doc ? s[n][4 * g + 2] : kHidden;
          s[n][4 * g + 3] = d.w == me.doc ? s[n][4 * g + 3] : kHidden;
        }
    }
  }
}

// The base of a row's weights is its running maximum itself, not a bound moved now and then: a row's largest
// weight is then 1, which bfloat16 rounds exactly (with a base up to 2^8 behind, attn_prompt_bf16 is 3% faster and
// its output 0.0020 of its size off, not 0.0018).
// Softmax weights of N score blocks; true (in every lane of the wave) if sums made before have to
// be multiplied by alpha. (Scores are rounded before the base is taken off, never fused with it: the largest one's
// weight is then 2^0 at any size of the scores.)
template <bool U, int N>
__device__ __forceinline__ bool weigh(v16f (&s)[N], const Params& p, Running& r, float& alpha) {
#pragma clang fp contract(off)
  float top = s[0][0];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = U ? fminf(top, s[n][i]) : fmaxf(top, s[n][i]);
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
  top = U ? fminf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) : fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  const float cap2 = p.to_score2;
  if (U) top = fmaf(-2.f * cap2, top, cap2);
  const bool move = top > r.m;
  const bool any = __any(move);
  if (any) {
    const float m = move ? top : r.m;
    alpha = r.m == kNegInf ? 0.f : fast_exp2(r.m - m);
    r.m = m;
    r.l *= alpha;
  }
  const float base = r.m == kNegInf ? 0.f : r.m;  // nothing seen yet: every weight is 2^-inf
  const float a = U ? cap2 - base : -base;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[n][i] = fast_exp2(U ? fmaf(-2.f * cap2, s[n][i], a) : s[n][i] + a);
  return any;
}

// The weights' sum, of the rounded ones where the products take rounded ones: numerator and denominator
// of the mean then err together.
__device__ __forceinline__ void add_weights(const Frag<1>& w, const v16f&, int, float& l) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 one = __builtin_bit_cast(bf16x2, 0x3f803f80u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = w.p[0][i];  // a copy: a bit cast of the vector's element reads its first one
    l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), one, l, false);
  }
}
__device__ __forceinline__ void add_weights(const Frag<3>&, const v16f& s, int half, float& l) {
#pragma unroll
  for (int i = 0; i < 8; ++i) l += s[8 * half + i];
}

// Four consecutive outputs, and what their rounding left out where that is wanted.
template <int PARTS>
__device__ __forceinline__ void store_out(const Params& p, int64_t off, float a, float b, float c, float d) {
  store_four<PARTS>(p.out, off, a, b, c, d);
  if constexpr (PARTS == 1) {
    if (p.out_low != nullptr) {
      auto low = [](float x) { return x - bf16_to_f32(f32_to_bf16(x)); };
      store_four<PARTS>(p.out_low, off, low(a), low(b), low(c), low(d));
    }
  }
}

// Divided keys: partial [rows of (b, i, h)][parts][D] sums and stats [..][parts][2] (base, sum).
struct Parts {
  float *partial, *stats;
  int n;  // 1: not divided, the results go to out and lse
};

template <int DP, int PARTS, bool CAP, bool SLOPE>
__global__ void __launch_bounds__(kThreads, PARTS == 1 || DP <= 64 ? 2 : 1) token_fwd_kernel(Params p, const DocTile* doc_tiles, Parts parts) {
  constexpr int KB = kKeys<DP, PARTS>, NB = KB / 32, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = KB * CH / kThreads, STEP = kThreads / CH;  // of the copies through registers
  constexpr int BUFS = PARTS == 1 ? 2 : 1;
  constexpr bool U = CAP && !SLOPE && PARTS == 1;
  typedef Tile<KB, DP, PARTS> KV;
  // two buffers by name: the compiler has to see that a copy into one does not change what is read from the other
  __shared__ __align__(16) uint16_t k_lds0[KV::kPlane * PARTS], v_lds0[KV::kPlane * PARTS];
  __shared__ __align__(16) uint16_t k_lds1[PARTS == 1 ? KV::kPlane : 8], v_lds1[PARTS == 1 ? KV::kPlane : 8];
  __shared__ __align__(16) int doc_lds[BUFS][KB];
  __shared__ int range_lds[4][2];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  const int tiles = (p.Nq + kQB - 1) / kQB;
  const Unit unit(p, blockIdx.x, p.G * parts.n, tiles, true, p.q_order);  // the longest rows of a causal mask first
  const int part = unit.inner % parts.n, g = unit.inner / parts.n;
  const int q0 = unit.tile * kQB, hk = unit.hk, b = unit.b, h = hk * p.G + g;
  const int n = kv_length(p, b);

  const int i = q0 + 32 * wave + c, row = i < p.Nq ? i : p.Nq - 1;
  const Sight me(p, b, row, n);
  const float slope2 = SLOPE ? p.slopes[h] * kLog2e : 0.f;
  const int wave_first = __builtin_amdgcn_readfirstlane(me.last);
  const int wave_last = __builtin_amdgcn_readlane(me.last, 31);
  // keys that any query of the workgroup may see: the last query's
  const int keys = Sight(p, b, min(q0 + kQB, p.Nq) - 1, n).last + 1;
  const bool by_document = p.documents != nullptr;
  int wave_lo = 0, wave_hi = 0, lo = 0, hi = 0;
  bool one_document = false;
  if (by_document) {
    document_range(me.doc, wave_lo, wave_hi);
    one_document = wave_lo == wave_hi && !__any(me.doc < 0);
    if (lane == 0) range_lds[wave][0] = wave_lo, range_lds[wave][1] = wave_hi;
    __syncthreads();
    lo = min(min(range_lds[0][0], range_lds[1][0]), min(range_lds[2][0], range_lds[3][0]));
    hi = max(max(range_lds[0][1], range_lds[1][1]), max(range_lds[2][1], range_lds[3][1]));
  }
  const DocTile* const row_tiles = doc_tiles + static_cast<int64_t>(b) * ((p.Nk + kDocTile - 1) / kDocTile);
  auto range = [row_tiles](int t) { return row_tiles[t * KB / kDocTile]; };
  Walk<decltype(range)> walk(0, keys > 0 ? (keys + KB - 1) / KB : 0, by_document, lo, hi, range);
  if (parts.n > 1) walk.take_part(part, parts.n, lane);
  const int end = walk.end;

  Frag<PARTS> q[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> r;
    const int d = 16 * s + 8 * hh;
    r.load(p.q.data, b * p.q.batch + row * p.q.token + h * p.q.head + d, d < p.D);
    q[s] = frag(r);
  }
  v16f o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = v16f{};
  Running run;

  const Copy<KB, DP> copy_k(p.k, b, hk, p.D, tid), copy_v(p.v, b, hk, p.D, tid);
  const int lr = tid / CH, lc = tid % CH;
  Raw8<PARTS> rk[PARTS == 3 ? LOADS : 1], rv[PARTS == 3 ? LOADS : 1];
  int rdoc = -1;  // as loaded: waited for where it is used
  auto load = [&](int t, auto to) __attribute__((always_inline)) {
    const int k0 = t * KB;
    if (by_document && tid < KB) rdoc = k0 + tid < n ? p.documents[static_cast<int64_t>(b) * p.Nk + k0 + tid] : -1;
    if constexpr (PARTS == 1) {
      copy_k(to.value == 0 ? k_lds0 : k_lds1, k0, n);
      copy_v(to.value == 0 ? v_lds0 : v_lds1, k0, n);
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int key = k0 + lr + STEP * j;
        bool on = key < n && 8 * lc < p.D;
        rk[j].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + 8 * lc, on);
        if (by_document && on) on = key_document(p, b, key) >= 0;  // padding may hold anything
        rv[j].load(p.v.data, b * p.v.batch + key * p.v.token + hk * p.v.head + 8 * lc, on);
      }
    }
  };
  DocTile here{}, there{};
  int t = walk.next(walk.begin, lane, here);
  if (t < end) load(t, std::integral_constant<int, 0>{});
  // one tile, in buffer B
  auto step = [&](auto which) __attribute__((always_inline)) {
    constexpr int B = which.value;
    const KV kt{B == 0 ? k_lds0 : k_lds1}, vt{B == 0 ? v_lds0 : v_lds1};
    if (by_document && PARTS == 1 && tid < KB) doc_lds[B][tid] = max(rdoc, -1);
    if constexpr (PARTS == 1) copies_done();
    __syncthreads();
    if constexpr (PARTS == 3) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        kt.put(lr + STEP * j, lc, frag(rk[j]));
        vt.put(lr + STEP * j, lc, frag(rv[j]));
      }
      if (by_document && tid < KB) doc_lds[0][tid] = max(rdoc, -1);
      __syncthreads();
    } else if (by_document && here.pad) {  // padding may hold anything: its value rows become zeros
      constexpr int each = kThreads / KB;
      const int r = tid / each;
      if (doc_lds[B][r] < 0)
        for (int ch = tid % each; ch < CH; ch += each) vt.put(r, ch, Frag<PARTS>{});
      __syncthreads();
    }
    const int after = walk.next(t + 1, lane, there);
    if (after < end) load(after, std::integral_constant<int, BUFS == 2 ? 1 - B : 0>{});
    const int k0 = t * KB;
    const bool unseen = k0 > wave_last || (by_document && (here.lo > wave_hi || here.hi < wave_lo));
    if (!unseen) {
      // decided ahead of the products: see token_device.h on branches between a product and its first use
      const bool mixed = by_document && !(one_document && here.lo == here.hi && here.lo == wave_lo && !here.pad);
      const bool masked = mixed || k0 + KB - 1 > wave_first;
      v16f s[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = v16f{};
      ahead<DP / 16 * NB, PARTS>([&](int i) { return kt.rows(32 * (i % NB), i / NB, lane); },
                          [&](int i, const Frag<PARTS>& x) { s[i % NB] = mma(x, q[i / NB], s[i % NB]); });
      settle(s);
      scores<PARTS, CAP, SLOPE, U>(s, p, me, slope2, k0, hh, masked, mixed ? doc_lds[B] : nullptr);
      float alpha = 1.f;
      if (weigh<U>(s, p, run, alpha)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      }
      Frag<PARTS> w[2 * NB];
#pragma unroll
      for (int st = 0; st < 2 * NB; ++st) {
        w[st] = frag_of<PARTS>(s[st / 2], st % 2);
        add_weights(w[st], s[st / 2], st % 2, run.l);
      }
      ahead<2 * NB * DT, PARTS>([&](int i) { return vt.columns(16 * (i / DT), i % DT, lane); },
                         [&](int i, const Frag<PARTS>& x) { o[i % DT] = mma(x, w[i / DT], o[i % DT]); });
    }
    t = after;
    here = there;
  };
  while (t < end) {
    step(std::integral_constant<int, 0>{});
    if constexpr (BUFS == 2) {
      if (t < end) step(std::integral_constant<int, 1>{});
    }
  }
  settle(o);
  const float l = xor32_pair_sum(run.l);
  if (i >= p.Nq) return;
  const int64_t at = (static_cast<int64_t>(b) * p.Nq + i) * p.H + h;
  if (parts.n > 1) {
    const int64_t to = at * parts.n + part;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = 32 * dt + 8 * x + 4 * hh;
        if (d < p.D)
          *reinterpret_cast<v4f*>(parts.partial + to * p.D + d) =
              v4f{o[dt][4 * x], o[dt][4 * x + 1], o[dt][4 * x + 2], o[dt][4 * x + 3]};
      }
    if (hh == 0) parts.stats[to * 2] = run.m, parts.stats[to * 2 + 1] = l;
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = 32 * dt + 8 * x + 4 * hh;
      if (d < p.D)
        store_out<PARTS>(p, at * p.D + d, o[dt][4 * x] * inv, o[dt][4 * x + 1] * inv, o[dt][4 * x + 2] * inv,
                         o[dt][4 * x + 3] * inv);
    }
  if (p.lse != nullptr && hh == 0) p.lse[at] = l == 0.f ? kNegInf : (run.m + log2f(l)) * kLn2;
}

// Few queries: column pr of the products is query pr / G, head hk G + pr % G; CB blocks of 16 columns. Runs of `chunk`
// keys, one a wave, 32 keys at a time on v_mfma_f32_16x16x32_bf16 (token_device.h's layouts with 16-lane groups g: a
// lane's weights belong to keys 16 (j / 4) + 4 g + j % 4). Keys go from memory into the products' registers, values
// through LDS of the wave's own; each is loaded again as soon as its registers are free, so about 32 rows of
// each are in flight a wave all the time.
template <int DP, int PARTS, bool CAP, int CB>
__global__ void __launch_bounds__(kThreads, PARTS == 1 ? 2 : 1) token_few_kernel(Params p, int chunk, Parts parts) {
  constexpr int DS = DP / 32, DT = DP / 16, CH = DP / 8, LOADS = 32 * CH / 64, STEP = 64 / CH;
  typedef Tile<32, DP, PARTS> V;
  __shared__ __align__(16) uint16_t v_lds[4][V::kPlane * PARTS];
  __shared__ __align__(16) int doc_lds[4][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const V vt{v_lds[wave]};
  const int per = (parts.n + 3) / 4;
  int64_t id = blockIdx.x;
  const int run_id = 4 * static_cast<int>(id % per) + wave;
  id /= per;
  const int hk = static_cast<int>(id % p.Hk), b = static_cast<int>(id / p.Hk);
  const int n = kv_length(p, b);
  const int64_t first64 = static_cast<int64_t>(run_id) * chunk;
  if (run_id >= parts.n || first64 >= n) return;  // waves share nothing: no barriers
  const int first = static_cast<int>(first64), stop = min(n, first + chunk);
  const bool by_document = p.documents != nullptr;
  const int rows = p.Nq * p.G;
  Frag<PARTS> q[CB][DS];
  Sight me[CB] = {};
  float slope2[CB];
  int64_t at[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const int pr = min(16 * cb + c, rows - 1), i = pr / p.G, h = hk * p.G + pr % p.G;
    me[cb] = Sight(p, b, i, n);
    slope2[cb] = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
    at[cb] = ((static_cast<int64_t>(b) * p.Nq + i) * p.H + h) * parts.n + run_id;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      Raw8<PARTS> r;
      const int d = 32 * s + 8 * g;
      r.load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + d, d < p.D);
      q[cb][s] = frag(r);
    }
  }
  v4f o[CB][DT];
  Running run[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[cb][dt] = zero4();

  const int lr = lane / CH, lc = lane % CH;
  Raw8<PARTS> rk[2][DS], rv[LOADS];
  int rdoc = -1;
  auto load_k = [&](int k0) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int64_t key = min(k0 + 16 * kb + c, n - 1);  // behind the end: a real row, hidden by the mask
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const int d = 32 * s + 8 * g;
        rk[kb][s].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + d, d < p.D);
      }
    }
  };
  auto load_v = [&](int k0) {
    if (by_document && lane < 32) rdoc = k0 + lane < n ? p.documents[static_cast<int64_t>(b) * p.Nk + k0 + lane] : -1;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int64_t key = min(k0 + lr + STEP * j, n - 1);
      bool on = 8 * lc < p.D;
      if (by_document && on) on = p.documents[static_cast<int64_t>(b) * p.Nk + key] >= 0;  // padding may hold anything
      rv[j].load(p.v.data, b * p.v.batch + key * p.v.token + hk * p.v.head + 8 * lc, on);
    }
  };
  load_v(first);
  load_k(first);
  for (int k0 = first; k0 < stop; k0 += 32) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) vt.put(lr + STEP * j, lc, frag(rv[j]));
    if (by_document && lane < 32) doc_lds[wave][lane] = max(rdoc, -1);
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
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    Frag<PARTS> w[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const int k1 = k0 + 4 * g;
      float x[8], top = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = k1 + 16 * (i / 4) + i % 4;
        x[i] = s[cb][i / 4][i % 4];
        x[i] = CAP ? tanh_of<PARTS>(x[i] * p.to_tanh) * p.to_score2 : x[i] * p.to_score2;
        if (slope2[cb] != 0.f) x[i] -= slope2[cb] * static_cast<float>(abs(me[cb].pos - key));
        x[i] = key <= me[cb].last ? x[i] : kNegInf;
      }
      if (by_document) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = doc_lds[wave][4 * g + 16 * (i / 4) + i % 4] == me[cb].doc ? x[i] : kNegInf;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
      top = group_max(top);
      Running& r = run[cb];
      if (__any(top > r.m)) {
        const float m = fmaxf(r.m, top), alpha = r.m == kNegInf ? 0.f : fast_exp2(r.m - m);
        r.m = m;
        r.l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[cb][dt] *= alpha;
      }
      const float base = r.m == kNegInf ? 0.f : r.m;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fast_exp2(x[i] - base);
      v16f y = v16f{};
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i];
      w[cb] = frag_of<PARTS>(y, 0);
      add_weights(w[cb], y, 0, r.l);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const Frag<PARTS> v = vt.columns16(dt, lane);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o[cb][dt] = mma16(v, w[cb], o[cb][dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  settle(o);
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float l = group_sum(run[cb].l);
    if (16 * cb + c < rows) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int d = 16 * dt + 4 * g;
        if (d < p.D) *reinterpret_cast<v4f*>(parts.partial + at[cb] * p.D + d) = o[cb][dt];
      }
      if (g == 0) {
        parts.stats[at[cb] * 2] = run[cb].m;
        parts.stats[at[cb] * 2 + 1] = l;
      }
    }
  }
}

// Half waves of a workgroup that joins parts.
template <int WAYS>
constexpr int kHalves = WAYS > 8 ? WAYS : 8;

// Joins the parts of one row of (b, i, h): WAYS half waves take a row's parts in turn, four elements a lane; a workgroup
// has kHalves / WAYS rows at a time. chunk: keys a part, of which those that begin behind the row's end were not
// written; 0: all parts were.
template <int PARTS, int WAYS>
__global__ void __launch_bounds__(32 * kHalves<WAYS>) token_join_kernel(Params p, int chunk, Parts parts) {
  constexpr int HALVES = kHalves<WAYS>;
  __shared__ __align__(16) float o_lds[HALVES][HZ_TOKEN_MAX_HEAD];
  __shared__ float l_lds[HALVES];
  const int64_t rows = static_cast<int64_t>(p.B) * p.Nq * p.H;
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5, way = half % WAYS, d = 4 * lane;
  for (int64_t at0 = static_cast<int64_t>(blockIdx.x) * (HALVES / WAYS); at0 < rows; at0 += static_cast<int64_t>(gridDim.x) * (HALVES / WAYS)) {
    const int64_t at = at0 + half / WAYS;
    float m = kNegInf, l = 0.f;
    v4f o = zero4();
    if (at < rows) {
      const int b = static_cast<int>(at / (static_cast<int64_t>(p.Nq) * p.H));
      const int used = chunk > 0 ? (kv_length(p, b) + chunk - 1) / chunk : parts.n;
      const float* const st = parts.stats + at * parts.n * 2;
#pragma unroll 4
      for (int r = lane; r < used; r += 32) m = fmaxf(m, st[2 * r]);
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
      const float base = m == kNegInf ? 0.f : m;
#pragma unroll 4
      for (int r = way; r < used; r += WAYS) {
        const float a = fast_exp2(st[2 * r] - base);
        l += a * st[2 * r + 1];
        if (d < p.D) o += a * *reinterpret_cast<const v4f*>(parts.partial + (at * parts.n + r) * p.D + d);
      }
    }
    if constexpr (WAYS > 1) {
      __syncthreads();
      *reinterpret_cast<v4f*>(&o_lds[half][d]) = o;
      if (lane == 0) l_lds[half] = l;
      __syncthreads();
      if (way != 0) continue;
#pragma unroll
      for (int x = 1; x < WAYS; ++x) {
        l += l_lds[half + x];
        o += *reinterpret_cast<const v4f*>(&o_lds[half + x][d]);
      }
    }
    if (at >= rows) continue;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (d < p.D) store_out<PARTS>(p, at * p.D + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (p.lse != nullptr && lane == 0) p.lse[at] = l == 0.f ? kNegInf : (m + log2f(l)) * kLn2;
  }
}

// The few-query kernel takes the calls whose rows of query and head fit the 32 columns of one product.
bool few(const hz_token_attention& a) { return a.Nq * (a.H / a.Hk) <= 32; }

// Keys a run: about 6144 waves in all, at least one block of 32 keys (attn_token_long_bf16: 265 us, 295 with a third of
// the waves, 270 with twice as many); heads up to 32, whose waves hold fewer registers, 8192 (32 rows of 4000 keys, 16 on 8
// heads of 32: 30 us, 35 with 6144).
int run_keys(const hz_token_attention& a) {
  const int64_t waves = a.D <= 32 ? 8192 : 6144, wanted = (a.B * a.Hk * a.Nk + waves - 1) / waves;
  return static_cast<int>(((wanted < a.Nk ? wanted : a.Nk) + 31) / 32 * 32);
}

int64_t blocks_of(const hz_token_attention& a) { return a.B * a.H * ((a.Nq + kQB - 1) / kQB); }

// Parts of a row's keys. Many queries: as many as 512 workgroups (two a CU) want, each of at least 128 keys
// (attn_train_both_f32's forward, 192 workgroups undivided: 90 us, 66 so and for 1024; where 512 need no division, 1024 would
// cost 13%, 2 x 2048 tokens of 16 bfloat16 heads of 128, causal: 67 us and 75).
int parts_of(const hz_token_attention& a) {
  if (few(a)) {
    const int c = run_keys(a);
    return static_cast<int>((a.Nk + c - 1) / c);
  }
  return share_of(blocks_of(a), a.Nk, 512);
}

int64_t parts_bytes(const hz_token_attention& a) {
  const int n = parts_of(a);
  return few(a) || n > 1 ? a.B * a.Nq * a.H * n * (a.D + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

template <int DP, int PARTS, bool CAP>
hipError_t run(const hz_token_attention& a, void* workspace, hipStream_t stream) {
  Params p = make_params(a);
  const int64_t rows = a.B * a.Nq * a.H;
  Parts parts{static_cast<float*>(workspace), nullptr, parts_of(a)};
  parts.stats = parts.partial + rows * parts.n * a.D;
  int chunk = 0;
  if (few(a)) {
    chunk = run_keys(a);
    const unsigned grid = static_cast<unsigned>(a.B * a.Hk * ((parts.n + 3) / 4));
    if (a.Nq * (a.H / a.Hk) <= 16)
      token_few_kernel<DP, PARTS, CAP, 1><<<grid, kThreads, 0, stream>>>(p, chunk, parts);
    else
      token_few_kernel<DP, PARTS, CAP, 2><<<grid, kThreads, 0, stream>>>(p, chunk, parts);
  } else {
    DocTile* const tiles = reinterpret_cast<DocTile*>(static_cast<char*>(workspace) + (parts_bytes(a) + 15) / 16 * 16);
    if (hipError_t err = launch_docs(a, p, false, tiles, stream); err != hipSuccess) return err;
    const unsigned grid = static_cast<unsigned>(blocks_of(a) * parts.n);
    if (p.slopes != nullptr)
      token_fwd_kernel<DP, PARTS, CAP, true><<<grid, kThreads, 0, stream>>>(p, tiles, parts);
    else
      token_fwd_kernel<DP, PARTS, CAP, false><<<grid, kThreads, 0, stream>>>(p, tiles, parts);
    if (parts.n == 1) return hipGetLastError();
  }
  // half waves a row: 162 parts of each of 36 rows take 8 us with 32 and 12 with 8, 47 parts of 512 rows 11 and 9
  const unsigned grid = static_cast<unsigned>(rows < 65536 ? rows : 65536);
  if (parts.n <= 8)
    token_join_kernel<PARTS, 1><<<static_cast<unsigned>(rows < 8 * 65536 ? (rows + 7) / 8 : 65536), kThreads, 0, stream>>>(p, chunk, parts);
  else if (parts.n <= 64)
    token_join_kernel<PARTS, 8><<<grid, kThreads, 0, stream>>>(p, chunk, parts);
  else
    token_join_kernel<PARTS, 32><<<grid, 1024, 0, stream>>>(p, chunk, parts);
  return hipGetLastError();
}

}  // namespace

int64_t token_attention_fwd_workspace(const hz_token_attention& a) {
  const int64_t parts = (parts_bytes(a) + 15) / 16 * 16;
  return few(a) ? parts : parts + doc_bytes(a);
}

hipError_t launch_token_attention_fwd(const hz_token_attention& a, void* workspace, hipStream_t stream) {
  auto by_type = [&](auto dp) {
    constexpr int DP = dp.value;
    if (a.dtype == HZ_DTYPE_BF16)
      return a.softcap > 0.f ? run<DP, 1, true>(a, workspace, stream) : run<DP, 1, false>(a, workspace, stream);
    return a.softcap > 0.f ? run<DP, 3, true>(a, workspace, stream) : run<DP, 3, false>(a, workspace, stream);
  };
  if (a.D <= 32) return by_type(std::integral_constant<int, 32>{});
  if (a.D <= 64) return by_type(std::integral_constant<int, 64>{});
  return by_type(std::integral_constant<int, 128>{});
}

}  // namespace hz
