// Reverse mode of the token attention (formulas and masks: include/hz_token.h; operand layouts:
// token_device.h).
//
// Two kernels, each with its sums in registers, so that nothing is added atomically: one owns queries and
// streams keys (dq, and rowsum(dout out) for the other), one owns keys and streams the queries of
// every head that shares them (dk, dv). Both rebuild P = exp(s - lse) from the forward's lse (far from zero, from the
// row's largest score and sum, which the first forms again), so scores and dP are formed twice: nine products a tile
// pair (two for the score gradients' second bfloat16 part) where one kernel with atomic dq sums would need seven. Bound by
// the products and, between them, the exponentials' vector work; attn_train_packed_bf16 (8192 tokens in four documents, 16
// on 4 heads of 128): 220 us for dq, 354 for dk and dv, matrix cores busy 34% and 25%. Tiles are copied, skipped and masked as in the forward.
#include "token_device.h"

namespace hz {
namespace {

using namespace token;

constexpr int kBlock = kOrderBlock;  // queries (dq) or keys (dk, dv) a workgroup, 32 a wave

// Rows of a streamed tile: two tensors, float32 ones in three parts.
template <int DP, int PARTS>
constexpr int kRows = (DP == 128 && PARTS == 3) ? 32 : 64;

// What the exponent of a row's weights begins with: a score has its row's largest one, or lse2 (the logarithm of their
// sum, all in base 2), taken off. bfloat16, capped, no distance bias: with u = 1 / (1 + e^2y), tanh y = 1 - 2 u, and the
// score cap2 - 2 cap2 u has that taken off in one fused operation.
template <int PARTS, bool CAP, bool SLOPE>
constexpr bool kFused = CAP && PARTS == 1 && !SLOPE;
template <int PARTS, bool CAP, bool SLOPE>
__device__ __forceinline__ float row_base(const Params& p, float top2) {
  return (kFused<PARTS, CAP, SLOPE> ? p.to_score2 : 0.f) - top2;
}

// Exponent (base 2) of one pair's weight from its dot product x and the distance between query and key, and the cap's
// derivative g. A score is rounded before the row's base is added, never fused with it: the largest score of a row whose
// base it is then gives 2^0, however large it is, and so it is in every kernel that forms it. (Fused scores are at
// most 8192 log2 e: off by 2^-10 there.) bfloat16, capped: the derivative 4 u (1 - u) leaves its 4 to the end (grad_scale).
template <int PARTS, bool CAP, bool SLOPE>
__device__ __forceinline__ float exponent(const Params& p, float x, float slope2, float distance, float base, float& g) {
#pragma clang fp contract(off)
  float s;
  if constexpr (CAP && PARTS == 1) {
    const float u = __builtin_amdgcn_rcpf(1.f + fast_exp2(x * p.to_exp2));
    g = fmaf(-u, u, u);
    s = fmaf(-2.f * p.to_score2, u, SLOPE ? p.to_score2 : base);
    if constexpr (!SLOPE) return s;
  } else if constexpr (CAP) {
    const float t = tanh_of<PARTS>(x * p.to_tanh);
    g = fmaf(-t, t, 1.f);
    s = t * p.to_score2;
  } else {
    g = 1.f;
    s = x * p.to_score2;
  }
  if constexpr (SLOPE) s = fmaf(-slope2, fabsf(distance), s);
  return s + base;
}

// Weight and score gradient of one pair. The weight is at most 1: rebuilt from a rounded logarithm it comes out above 1 by
// that rounding.
template <int PARTS, bool CAP, bool SLOPE>
__device__ __forceinline__ void pair(const Params& p, float x, float dp, float slope2, float distance, float base,
                                     float delta, float& w, float& ds) {
  float g;
  w = lse_weight(exponent<PARTS, CAP, SLOPE>(p, x, slope2, distance, base, g));
  ds = w * (dp - delta);
  if constexpr (CAP) ds *= g;
}

// lse is a rounded logarithm, and its change of base rounds again: a weight rebuilt from it is off by up to five times
// 2^-24 |lse| of itself, all of a row's by the same factor. Rows whose lse is above this (or is not finite) get their largest
// score and their sum formed again, from the scores as the reverse pass forms them: weights 2^(s - m) / l. Below it they are
// off by 1e-5 (float32) and 8e-5 (bfloat16) at most; without it a lone key's weight was off by up to 1.4e-3 at a score of
// 10^4, 16% at 10^6, and NaN at 10^10. Where every block has such a row the reverse pass takes a quarter to a third longer (4 x
// 2048 tokens of 16 on 4 bfloat16 heads of 64: 250 us and 356; float32, 4 x 1024: 213 and 273), and twice as long
// where the keys are divided, since each part goes over all of them.
template <int PARTS>
constexpr float kFar = PARTS == 1 ? 256.f : 32.f;

// What dk, dv need of a query: the base of its weights' exponents (-inf: it sees nothing), rowsum(dout out), and
// what its weights are multiplied by (1 where the base holds their sum).
struct RowStats {
  float base, delta, inv, unused;
};
// Operands that are read together.
template <int PARTS>
struct Two {
  Frag<PARTS> a, b;
};
template <int PARTS>
struct Three {
  Frag<PARTS> a, b, c;
};

template <int PARTS, bool CAP>
__device__ __forceinline__ float grad_scale(const Params& p) {
  return CAP && PARTS == 1 ? 4.f * p.scale : p.scale;
}

// Sums made by several workgroups: `n` shares, partial [n][tensors][elements] in float32 for a last kernel to add up.
struct Splits {
  float* partial;
  int64_t elements;
  int n;      // 1: not divided, the results go where they belong
  int heads;  // of dk, dv: shares of the query heads; n / heads parts of the queries
};

template <int DP, int PARTS, bool CAP, bool SLOPE>
__global__ void __launch_bounds__(256, PARTS == 1 || DP <= 64 ? 2 : 1) token_dq_kernel(Params p, hz_token_tensor dout, void* dq,
                                                                           RowStats* stats, const DocTile* doc_tiles,
                                                                                      Splits splits) {
  constexpr int KB = kRows<DP, PARTS>, NB = KB / 32, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = KB * CH / 256, STEP = 256 / CH;
  constexpr int BUFS = PARTS == 1 ? 2 : 1;
  typedef Tile<KB, DP, PARTS> KV;
  __shared__ __align__(16) uint16_t k_lds0[KV::kPlane * PARTS], v_lds0[KV::kPlane * PARTS];
  __shared__ __align__(16) uint16_t k_lds1[PARTS == 1 ? KV::kPlane : 8], v_lds1[PARTS == 1 ? KV::kPlane : 8];
  __shared__ __align__(16) int doc_lds[BUFS][KB];
  __shared__ int range_lds[4][2];
  __shared__ int far_lds[4];
  __shared__ float inv_lds[kBlock];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  const int tiles = (p.Nq + kBlock - 1) / kBlock;
  const Unit unit(p, blockIdx.x, p.G * splits.n, tiles, true, p.q_order);  // the longest rows of a causal mask first
  const int part = unit.inner % splits.n;
  const int q0 = unit.tile * kBlock, hk = unit.hk, b = unit.b, h = hk * p.G + unit.inner / splits.n;
  const int n = kv_length(p, b);
  const int i = q0 + 32 * wave + c, row = i < p.Nq ? i : p.Nq - 1;
  const int64_t at = (static_cast<int64_t>(b) * p.Nq + row) * p.H + h;
  const float lse = p.lse[at];
  const bool far = !(fabsf(lse) <= kFar<PARTS>) && lse != kNegInf;
  const Sight me(p, b, row, n);
  const float slope2 = SLOPE ? p.slopes[h] * kLog2e : 0.f;
  const int wave_first = __builtin_amdgcn_readfirstlane(me.last);
  const int wave_last = __builtin_amdgcn_readlane(me.last, 31);
  const int keys = Sight(p, b, min(q0 + kBlock, p.Nq) - 1, n).last + 1;
  const bool by_document = p.documents != nullptr;
  int wave_lo = 0, wave_hi = 0, lo = 0, hi = 0;
  bool one_document = false;
  if (by_document) {
    document_range(me.doc, wave_lo, wave_hi);
    one_document = wave_lo == wave_hi && !__any(me.doc < 0);
    if (lane == 0) range_lds[wave][0] = wave_lo, range_lds[wave][1] = wave_hi;
  }
  const bool wave_far = __any(far);
  if (lane == 0) far_lds[wave] = wave_far;
  __syncthreads();
  if (by_document) {
    lo = min(min(range_lds[0][0], range_lds[1][0]), min(range_lds[2][0], range_lds[3][0]));
    hi = max(max(range_lds[0][1], range_lds[1][1]), max(range_lds[2][1], range_lds[3][1]));
  }
  const bool any_far = (far_lds[0] | far_lds[1] | far_lds[2] | far_lds[3]) != 0;
  const DocTile* const row_tiles = doc_tiles + static_cast<int64_t>(b) * ((p.Nk + kDocTile - 1) / kDocTile);
  auto range = [row_tiles](int t) { return row_tiles[t * KB / kDocTile]; };
  Walk<decltype(range)> walk(0, keys > 0 ? (keys + KB - 1) / KB : 0, by_document, lo, hi, range);

  Frag<PARTS> q[DP / 16], go[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> r;
    const int d = 16 * s + 8 * hh;
    r.load(p.q.data, b * p.q.batch + row * p.q.token + h * p.q.head + d, d < p.D);
    q[s] = frag(r);
  }
  const Copy<KB, DP> copy_k(p.k, b, hk, p.D, tid), copy_v(p.v, b, hk, p.D, tid);
  const int lr = tid / CH, lc = tid % CH;
  float base = row_base<PARTS, CAP, SLOPE>(p, lse == kNegInf ? 0.f : lse * kLog2e);  // -inf: a row that sees nothing
  if (hh == 0) inv_lds[32 * wave + c] = 1.f;
  if (any_far) {
    // The rows' largest scores m and sums l of 2^(s - m), over all keys that they see (kFar): the scores' part of the loop
    // below with the softmax's running maximum, one tile at a time.
    const KV kt{k_lds0};
    Walk<decltype(range)> all = walk;
    DocTile here{};
    float m = kNegInf, l = 0.f;
    for (int t = all.next(all.begin, lane, here); t < all.end; t = all.next(t + 1, lane, here)) {
      const int k0 = t * KB;
      if (by_document && tid < KB) doc_lds[0][tid] = k0 + tid < n ? key_document(p, b, k0 + tid) : -1;
      if constexpr (PARTS == 1) {
        copy_k(k_lds0, k0, n);
        copies_done();
      } else {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const int key = k0 + lr + STEP * j;
          Raw8<PARTS> r;
          r.load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + 8 * lc, key < n && 8 * lc < p.D);
          kt.put(lr + STEP * j, lc, frag(r));
        }
      }
      __syncthreads();
      if (k0 <= wave_last) {
#pragma unroll 1
        for (int nb = 0; nb < NB; ++nb) {
          v16f s[1] = {v16f{}};
#pragma unroll
          for (int ds = 0; ds < DP / 16; ++ds) s[0] = mma(kt.rows(32 * nb, ds, lane), q[ds], s[0]);
          settle(s);
          const int k1 = k0 + 32 * nb + 4 * hh;
          const float away = static_cast<float>(me.pos - k1);
          float top = kNegInf;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float g;
            const float y = exponent<PARTS, CAP, SLOPE>(p, s[0][e], slope2, away - static_cast<float>(row_of(e, 0)),
                                                        row_base<PARTS, CAP, SLOPE>(p, 0.f), g);
            const bool seen = row_of(e, 0) <= me.last - k1 &&
                              (!by_document || doc_lds[0][32 * nb + 4 * hh + row_of(e, 0)] == me.doc);
            top = seen ? fmaxf(top, y) : top;
          }
          const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
          top = fmaxf(m, fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
          l *= m == kNegInf ? 0.f : fast_exp2(m - top);
          m = top;
          const float from = row_base<PARTS, CAP, SLOPE>(p, m == kNegInf ? 0.f : m);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float g;
            const float y = exponent<PARTS, CAP, SLOPE>(p, s[0][e], slope2, away - static_cast<float>(row_of(e, 0)), from, g);
            const bool seen = row_of(e, 0) <= me.last - k1 &&
                              (!by_document || doc_lds[0][32 * nb + 4 * hh + row_of(e, 0)] == me.doc);
            // (a NaN, or a score of +inf, makes a NaN of the sum, and so of all of the row's weights)
            l += seen ? (y > 0.f ? 1.f : fast_exp2(y)) : 0.f;
          }
        }
      }
      __syncthreads();
    }
    l = xor32_pair_sum(l);
    if (far && l != 0.f) {
      base = l == l ? row_base<PARTS, CAP, SLOPE>(p, m) : l;
      if (hh == 0) inv_lds[32 * wave + c] = 1.f / l;
    }
  }
  if (splits.n > 1) walk.take_part(part, splits.n, lane);
  const int end = walk.end;

  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> rg, ro;
    const int d = 16 * s + 8 * hh;
    rg.load(dout.data, b * dout.batch + row * dout.token + h * dout.head + d, d < p.D);
    ro.load(p.out, at * p.D + d, d < p.D);
    float x[8], y[8];
    floats(rg, x);
    floats(ro, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += x[j] * y[j];
    if (PARTS == 1 && p.out_low != nullptr) {
      ro.load(p.out_low, at * p.D + d, d < p.D);
      floats(ro, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += x[j] * y[j];
    }
    go[s] = frag(rg);
  }
  delta = xor32_pair_sum(delta);
  if (i < p.Nq && hh == 0 && part == 0)
    *reinterpret_cast<float4*>(stats + at) = make_float4(lse == kNegInf ? kNegInf : base, delta, inv_lds[32 * wave + c], 0.f);
  v16f acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = v16f{};

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
        if (by_document && on) on = key_document(p, b, key) >= 0;  // padding may hold anything
        rk[j].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + 8 * lc, on);
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
    } else if (by_document && here.pad) {  // padding may hold anything: its rows become zeros
      constexpr int each = 256 / KB;
      const int r = tid / each;
      if (doc_lds[B][r] < 0)
        for (int ch = tid % each; ch < CH; ch += each) kt.put(r, ch, Frag<PARTS>{}), vt.put(r, ch, Frag<PARTS>{});
      __syncthreads();
    }
    const int after = walk.next(t + 1, lane, there);
    if (after < end) load(after, std::integral_constant<int, BUFS == 2 ? 1 - B : 0>{});
    const int k0 = t * KB;
    const bool unseen = k0 > wave_last || (by_document && (here.lo > wave_hi || here.hi < wave_lo));
    if (!unseen) {
      const bool mixed = by_document && !(one_document && here.lo == here.hi && here.lo == wave_lo && !here.pad);
      const bool masked = mixed || k0 + KB - 1 > wave_first;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        v16f s = v16f{}, dp = v16f{};
        const int l = PARTS == 3 ? anew(lane) : lane;
        ahead<DP / 16, PARTS>([&](int ds) { return Two<PARTS>{kt.rows(32 * nb, ds, l), vt.rows(32 * nb, ds, l)}; },
                       [&](int ds, const Two<PARTS>& x) {
                         s = mma(x.a, q[ds], s);
                         dp = mma(x.b, go[ds], dp);
                       });
        const int k1 = k0 + 32 * nb + 4 * hh;
        const float away = static_cast<float>(me.pos - k1);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float w, g;
          pair<PARTS, CAP, SLOPE>(p, s[e], dp[e], slope2, away - static_cast<float>(row_of(e, 0)), base, delta, w, g);
          s[e] = g;
        }
        if (masked) {
          const int last = me.last - k1;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = row_of(e, 0) <= last ? s[e] : 0.f;
          if (mixed) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int4 d = *reinterpret_cast<const int4*>(&doc_lds[B][32 * nb + 8 * e + 4 * hh]);
              s[4 * e] = d.x == me.doc ? s[4 * e] : 0.f;
              s[4 * e + 1] = d.y == me.doc ? s[4 * e + 1] : 0.f;
              s[4 * e + 2] = d.z == me.doc ? s[4 * e + 2] : 0.f;
              s[4 * e + 3] = d.w == me.doc ? s[4 * e + 3] : 0.f;
            }
          }
        }
        Frag<PARTS == 1 ? 2 : 3> g;
        ahead<2 * DT, PARTS>([&](int i) { return kt.columns(32 * nb + 16 * (i / DT), i % DT, l); },
                      [&](int i, const Frag<PARTS>& x) {
                        if (i % DT == 0) g = grad_frag<PARTS>(s, i / DT);
                        acc[i % DT] = mma(x, g, acc[i % DT]);
                      });
      }
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
  settle(acc);
  if (i >= p.Nq) return;
  const float to_grad = grad_scale<PARTS, CAP>(p) * inv_lds[32 * wave + c];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = 32 * dt + 8 * x + 4 * hh;
      if (d >= p.D) continue;
      if (splits.n > 1)
        store_four<3>(splits.partial + part * splits.elements, at * p.D + d, acc[dt][4 * x] * to_grad, acc[dt][4 * x + 1] * to_grad,
                      acc[dt][4 * x + 2] * to_grad, acc[dt][4 * x + 3] * to_grad);
      else
        store_four<PARTS>(dq, at * p.D + d, acc[dt][4 * x] * to_grad, acc[dt][4 * x + 1] * to_grad,
                          acc[dt][4 * x + 2] * to_grad, acc[dt][4 * x + 3] * to_grad);
    }
}

// WAVES = 8: waves w and w + 4 own the same 32 keys and take the tile's first and second 32 queries; their sums meet in LDS
// at the end. So two waves share a SIMD although a workgroup owns 128 keys only (float32 heads of 64:
// attn_train_both_f32 269 us with four waves, 234 with eight). The values' rows are in LDS, and the keys' too where
// there are not the registers for them: float32, and bfloat16 heads of 128, where it saves the spilling of addresses
// (attn_train_packed_bf16 814 -> 798 us); heads of 64 and 32 keep them in registers (1% and 2% faster).
template <int DP, int PARTS, bool CAP, bool SLOPE, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, WAVES == 8 || DP <= 32 ? 2 : 1) token_dkv_kernel(Params p, hz_token_tensor dout, const RowStats* stats,
                                                                          void* dk, void* dv, const DocTile* doc_tiles, Splits splits) {
  constexpr int THREADS = 64 * WAVES, SETS = WAVES / 4;
  constexpr int QB = kRows<DP, PARTS>, NB = QB / 32 / SETS, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = QB * CH / THREADS, STEP = THREADS / CH;
  constexpr int BUFS = PARTS == 1 ? 2 : 1;
  constexpr bool KEYS_IN_LDS = WAVES == 8 && (PARTS == 3 || DP == 128);
  typedef Tile<QB, DP, PARTS> QT;
  __shared__ __align__(16) uint16_t q_lds0[QT::kPlane * PARTS], g_lds0[QT::kPlane * PARTS];
  __shared__ __align__(16) uint16_t q_lds1[PARTS == 1 ? QT::kPlane : 8], g_lds1[PARTS == 1 ? QT::kPlane : 8];
  __shared__ __align__(16) float base_lds[BUFS][QB], delta_lds[BUFS][QB], inv_lds[BUFS][QB];
  __shared__ __align__(16) int doc_lds[BUFS][QB];
  __shared__ __align__(16) uint16_t v_lds[kBlock * DP * PARTS];
  __shared__ __align__(16) uint16_t k_lds[KEYS_IN_LDS ? kBlock * DP * PARTS : 8];
  __shared__ uint64_t bad_lds[BUFS], scaled_lds[BUFS];
  __shared__ int range_lds[4][2];
  const int tid = threadIdx.x, wave = (tid >> 6) & 3, set = tid >> 8, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  // the first keys of a causal mask are seen by the most queries
  const Unit unit(p, blockIdx.x, splits.n, (p.Nk + kBlock - 1) / kBlock, false, p.k_order);
  const int key0 = unit.tile * kBlock, hk = unit.hk, b = unit.b;
  const int share = unit.inner / (splits.n / splits.heads), part = unit.inner % (splits.n / splits.heads);
  const int first_head = share * p.G / splits.heads, last_head = (share + 1) * p.G / splits.heads - 1;
  const int n = kv_length(p, b), shift = n - p.Nq;  // position of query 0
  const int wave0 = key0 + 32 * wave, key = wave0 + c, row = key < n ? key : max(n - 1, 0);
  const int prefix = p.causal && p.prefix != nullptr ? p.prefix[b] : 0;
  const bool always = !p.causal || key < prefix;  // seen from every position, else from `key` on
  const bool by_document = p.documents != nullptr;
  const int my_doc = by_document && key < n ? key_document(p, b, key) : -1;
  int wave_lo = 0, wave_hi = 0, lo = 0, hi = 0;
  bool one_document = false;
  if (by_document) {
    document_range(my_doc, wave_lo, wave_hi);
    one_document = wave_lo == wave_hi && !__any(my_doc < 0);
    if (lane == 0) range_lds[wave][0] = wave_lo, range_lds[wave][1] = wave_hi;
    __syncthreads();
    lo = min(min(range_lds[0][0], range_lds[1][0]), min(range_lds[2][0], range_lds[3][0]));
    hi = max(max(range_lds[0][1], range_lds[1][1]), max(range_lds[2][1], range_lds[3][1]));
  }

  Frag<PARTS> k[KEYS_IN_LDS ? 1 : DP / 16];
  if constexpr (!KEYS_IN_LDS) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      Raw8<PARTS> rk;
      const int d = 16 * s + 8 * hh;
      rk.load(p.k.data, b * p.k.batch + row * p.k.token + hk * p.k.head + d, key < n && d < p.D);
      k[s] = frag(rk);
    }
  }
  const Tile<kBlock, DP, PARTS> vt{v_lds}, keys{k_lds};
  for (int i = tid; i < kBlock * CH; i += THREADS) {
    const int r = i / CH, ch = i % CH;
    Raw8<PARTS> rv;
    rv.load(p.v.data, b * p.v.batch + (key0 + r) * p.v.token + hk * p.v.head + 8 * ch, key0 + r < n && 8 * ch < p.D);
    vt.put(r, ch, frag(rv));
    if constexpr (KEYS_IN_LDS) {
      rv.load(p.k.data, b * p.k.batch + (key0 + r) * p.k.token + hk * p.k.head + 8 * ch, key0 + r < n && 8 * ch < p.D);
      keys.put(r, ch, frag(rv));
    }
  }
  v16f ak[DT], av[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ak[dt] = v16f{}, av[dt] = v16f{};

  // the tiles of queries that may see a key of this block
  const int begin = p.causal && key0 >= prefix ? max(0, key0 - shift) / QB : 0;
  const int doc_row = (p.Nk + kDocTile - 1) / kDocTile;
  const DocTile* const row_tiles = doc_tiles + static_cast<int64_t>(b) * doc_row;
  auto range = [row_tiles, shift, n](int t) {
    // the tile's queries stand at 64 or fewer consecutive positions, which meet at most two tiles of keys
    const int first = shift + t * QB, last = min(first + QB, n) - 1;
    if (last < 0) return DocTile{2147483647, -1, 1, 0};
    DocTile a = row_tiles[max(first, 0) / kDocTile];
    const DocTile z = row_tiles[last / kDocTile];
    return DocTile{min(a.lo, z.lo), max(a.hi, z.hi), a.pad | z.pad | (first < 0), 0};
  };
  Walk<decltype(range)> walk(begin, key0 < n ? (p.Nq + QB - 1) / QB : 0, by_document, lo, hi, range);
  if (splits.n > splits.heads) walk.take_part(part, splits.n / splits.heads, lane);
  const int end = walk.end;
  const int lr = tid / CH, lc = tid % CH;
  Raw8<PARTS> rq[PARTS == 3 ? LOADS : 1], rg[PARTS == 3 ? LOADS : 1];
  float4 rstat = make_float4(0.f, 0.f, 1.f, 0.f);  // as loaded: waited for where they are used
  int rdoc = 0;
  auto load = [&](int head, int t, auto to) __attribute__((always_inline)) {
    const int h = hk * p.G + head, q0 = t * QB;
    if (tid < QB) {
      const int i = min(q0 + tid, p.Nq - 1);
      rstat = *reinterpret_cast<const float4*>(stats + (static_cast<int64_t>(b) * p.Nq + i) * p.H + h);
      if (q0 + tid >= p.Nq) rstat.x = kNegInf;
      if (by_document) rdoc = shift + i >= 0 ? p.documents[static_cast<int64_t>(b) * p.Nk + shift + i] : -1;
    }
    if constexpr (PARTS == 1) {
      if (set == 0) {
        const Copy<QB, DP> copy(p.q, b, h, p.D, tid & 255);
        copy(to.value == 0 ? q_lds0 : q_lds1, q0, p.Nq);
      }
      if (set == SETS - 1) {
        const Copy<QB, DP> copy(dout, b, h, p.D, tid & 255);
        copy(to.value == 0 ? g_lds0 : g_lds1, q0, p.Nq);
      }
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int i = q0 + lr + STEP * j;
        bool on = i < p.Nq && 8 * lc < p.D;
        if (on) on = p.lse[(static_cast<int64_t>(b) * p.Nq + i) * p.H + h] != kNegInf;  // padding may hold anything
        rq[j].load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + 8 * lc, on);
        rg[j].load(dout.data, b * dout.batch + i * dout.token + h * dout.head + 8 * lc, on);
      }
    }
  };
  DocTile here{}, there{};
  int head = first_head, t = walk.next(walk.begin, lane, here);
  if (t < end) load(head, t, std::integral_constant<int, 0>{});
  // one tile of one head, in buffer B
  auto step = [&](auto which) __attribute__((always_inline)) {
    constexpr int B = which.value;
    const QT qt{B == 0 ? q_lds0 : q_lds1}, gt{B == 0 ? g_lds0 : g_lds1};
    auto put_rows = [&] {
      if (tid < QB) {
        // a query that sees nothing, or is none: weights of 2^-inf
        const bool bad = rstat.x == kNegInf;
        const uint64_t votes = __ballot(bad), scaled = __ballot(!bad && rstat.z != 1.f);
        base_lds[B][tid] = rstat.x;
        delta_lds[B][tid] = bad ? 0.f : rstat.y;
        inv_lds[B][tid] = rstat.z;
        if (by_document) doc_lds[B][tid] = rdoc >= 0 ? rdoc : kNoDocument;
        if (tid == 0) bad_lds[B] = votes, scaled_lds[B] = scaled;
      }
    };
    if constexpr (PARTS == 1) {
      put_rows();
      copies_done();
    }
    __syncthreads();
    if constexpr (PARTS == 3) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        qt.put(lr + STEP * j, lc, frag(rq[j]));
        gt.put(lr + STEP * j, lc, frag(rg[j]));
      }
      put_rows();
      __syncthreads();
    } else if (const uint64_t bad = bad_lds[B]; bad != 0) {  // such rows may hold anything: they become zeros
      constexpr int each = THREADS / QB;
      const int r = tid / each;
      if ((bad >> r) & 1)
        for (int ch = tid % each; ch < CH; ch += each) qt.put(r, ch, Frag<PARTS>{}), gt.put(r, ch, Frag<PARTS>{});
      __syncthreads();
    }
    int after = walk.next(t + 1, lane, there), next_head = head;
    if (after >= end && head < last_head) {
      next_head = head + 1;
      after = walk.next(walk.begin, lane, there);
    }
    if (after < end) load(next_head, after, std::integral_constant<int, BUFS == 2 ? 1 - B : 0>{});
    const int p0 = shift + t * QB;  // position of the tile's first query
    const float slope2 = SLOPE ? p.slopes[hk * p.G + head] * kLog2e : 0.f;
    const bool unseen = (p.causal && wave0 >= prefix && p0 + QB - 1 < wave0) ||
                        (by_document && (here.lo > wave_hi || here.hi < wave_lo));
    if (!unseen) {
      const bool mixed = by_document && !(one_document && here.lo == here.hi && here.lo == wave_lo && !here.pad);
      const bool masked = mixed || wave0 + 31 >= n || (p.causal && wave0 + 31 >= prefix && p0 < wave0 + 31);
      const bool scaled = scaled_lds[B] != 0;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int r0 = 32 * (nb + (SETS == 2 ? set : 0));
        v16f s = v16f{}, dp = v16f{};
        const int l = anew(lane);
        ahead<DP / 16, PARTS>(
            [&](int ds) { return Three<PARTS>{qt.rows(r0, ds, l), gt.rows(r0, ds, l), vt.rows(32 * wave, ds, l)}; },
            [&](int ds, const Three<PARTS>& x) {
              if constexpr (KEYS_IN_LDS)
                s = mma_turned(x.a, keys.rows(32 * wave, ds, l), s);
              else
                s = mma_turned(x.a, k[ds], s);
              dp = mma_turned(x.b, x.c, dp);
            });
        const int r1 = r0 + 4 * hh;
        const float away = static_cast<float>(p0 + r1 - key);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const v4f b0 = *reinterpret_cast<const v4f*>(&base_lds[B][r1 + 8 * e]);
          const v4f d = *reinterpret_cast<const v4f*>(&delta_lds[B][r1 + 8 * e]);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float w, gs;
            pair<PARTS, CAP, SLOPE>(p, s[4 * e + x], dp[4 * e + x], slope2, away + static_cast<float>(8 * e + x), b0[x], d[x], w, gs);
            s[4 * e + x] = w;
            dp[4 * e + x] = gs;
          }
        }
        if (scaled) {  // weights 2^(s - m) get their rows' 1 / l
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const v4f inv = *reinterpret_cast<const v4f*>(&inv_lds[B][r1 + 8 * e]);
#pragma unroll
            for (int x = 0; x < 4; ++x) s[4 * e + x] *= inv[x], dp[4 * e + x] *= inv[x];
          }
        }
        if (masked) {
          const int first = key >= n ? 32 : always ? 0 : key - p0 - r1;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool seen = row_of(e, 0) >= first;
            s[e] = seen ? s[e] : 0.f;
            dp[e] = seen ? dp[e] : 0.f;
          }
          if (mixed) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int4 d = *reinterpret_cast<const int4*>(&doc_lds[B][r1 + 8 * e]);
              const bool seen[4] = {d.x == my_doc, d.y == my_doc, d.z == my_doc, d.w == my_doc};
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                s[4 * e + x] = seen[x] ? s[4 * e + x] : 0.f;
                dp[4 * e + x] = seen[x] ? dp[4 * e + x] : 0.f;
              }
            }
          }
        }
        Frag<PARTS> w;
        Frag<PARTS == 1 ? 2 : 3> gs;
        ahead<2 * DT, PARTS>(
            [&](int i) { return Two<PARTS>{gt.columns(r0 + 16 * (i / DT), i % DT, l), qt.columns(r0 + 16 * (i / DT), i % DT, l)}; },
            [&](int i, const Two<PARTS>& x) {
              if (i % DT == 0) w = frag_of<PARTS>(s, i / DT), gs = grad_frag<PARTS>(dp, i / DT);
              av[i % DT] = mma(x.a, w, av[i % DT]);
              ak[i % DT] = mma(x.b, gs, ak[i % DT]);
            });
      }
    }
    t = after;
    head = next_head;
    here = there;
  };
  while (t < end) {
    step(std::integral_constant<int, 0>{});
    if constexpr (BUFS == 2) {
      if (t < end) step(std::integral_constant<int, 1>{});
    }
  }
  settle(ak);
  settle(av);
  if constexpr (SETS == 2) {
    // 16 accumulators a lane and round: what one tile buffer of queries and one of dout hold
    float* const to[2] = {reinterpret_cast<float*>(q_lds0), reinterpret_cast<float*>(g_lds0)};
    constexpr int each = QT::kBytes / (4 * 64 * 16);  // quadruples a lane that one buffer holds
    auto join = [&](v16f(&a)[DT]) {
#pragma unroll
      for (int r = 0; r < 4 * DT; r += 2 * each) {
        __syncthreads();
        if (set == 1) {
#pragma unroll
          for (int x = r; x < r + 2 * each && x < 4 * DT; ++x)
            *reinterpret_cast<v4f*>(to[(x - r) / each] + (((x - r) % each * 4 + wave) * 64 + lane) * 4) =
                v4f{a[x / 4][4 * (x % 4)], a[x / 4][4 * (x % 4) + 1], a[x / 4][4 * (x % 4) + 2], a[x / 4][4 * (x % 4) + 3]};
        }
        __syncthreads();
        if (set == 0) {
#pragma unroll
          for (int x = r; x < r + 2 * each && x < 4 * DT; ++x) {
            const v4f y = *reinterpret_cast<const v4f*>(to[(x - r) / each] + (((x - r) % each * 4 + wave) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[x / 4][4 * (x % 4) + e] += y[e];
          }
        }
      }
    };
    join(ak);
    join(av);
    if (set == 1) return;
  }
  if (key >= p.Nk) return;
  const int64_t at = ((static_cast<int64_t>(b) * p.Nk + key) * p.Hk + hk) * p.D;
  const float to_grad = grad_scale<PARTS, CAP>(p);
  if (splits.n > 1) {
    float* const to = splits.partial + unit.inner * 2 * splits.elements + at;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = 32 * dt + 8 * x + 4 * hh;
        if (d < p.D) {
          store_four<3>(to, d, ak[dt][4 * x] * to_grad, ak[dt][4 * x + 1] * to_grad, ak[dt][4 * x + 2] * to_grad,
                        ak[dt][4 * x + 3] * to_grad);
          store_four<3>(to + splits.elements, d, av[dt][4 * x], av[dt][4 * x + 1], av[dt][4 * x + 2], av[dt][4 * x + 3]);
        }
      }
    return;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = 32 * dt + 8 * x + 4 * hh;
      if (d < p.D) {
        store_four<PARTS>(dk, at + d, ak[dt][4 * x] * to_grad, ak[dt][4 * x + 1] * to_grad, ak[dt][4 * x + 2] * to_grad,
                          ak[dt][4 * x + 3] * to_grad);
        store_four<PARTS>(dv, at + d, av[dt][4 * x], av[dt][4 * x + 1], av[dt][4 * x + 2], av[dt][4 * x + 3]);
      }
    }
}

// Sums of the shares of one tensor, or of two of the same size, four elements a thread.
template <int PARTS>
__global__ void __launch_bounds__(256) token_sum_kernel(Splits splits, int tensors, void* first, void* second) {
  const int64_t quads = splits.elements / 4, all = tensors * quads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    v4f sum = *reinterpret_cast<const v4f*>(splits.partial + 4 * i);
#pragma unroll 4
    for (int s = 1; s < splits.n; ++s) sum += *reinterpret_cast<const v4f*>(splits.partial + 4 * (s * all + i));
    if (i < quads)
      store_four<PARTS>(first, 4 * i, sum[0], sum[1], sum[2], sum[3]);
    else
      store_four<PARTS>(second, 4 * (i - quads), sum[0], sum[1], sum[2], sum[3]);
  }
}

template <int PARTS>
void launch_sum(const Splits& splits, int tensors, void* first, void* second, hipStream_t stream) {
  if (splits.n == 1) return;
  const int64_t n = (tensors * splits.elements / 4 + 255) / 256;
  token_sum_kernel<PARTS><<<static_cast<unsigned>(n < 8192 ? n : 8192), 256, 0, stream>>>(splits, tensors, first, second);
}

// Workgroups are made more by dividing the keys (dq), the query heads of a key head and then the queries (dk, dv):
// documents and causal masks make them of very different lengths, which a single round of them cannot even out, and a
// few long sequences would leave most CUs idle. The sum of the shares costs little beside that
// (attn_train_packed_bf16 825 us in all, undivided 1097; attn_train_both_f32 262 and 434). For 1024 workgroups instead of 512
// the first would take 1% less, but 4 x 2048 tokens of 16 on 4 heads of 64 8% more (293 us, 316).
Splits dq_splits(const hz_token_attention& a) {
  const int64_t blocks = a.B * a.H * ((a.Nq + kBlock - 1) / kBlock);
  return {nullptr, a.B * a.Nq * a.H * a.D, share_of(blocks, a.Nk, 512), 1};
}

Splits dkv_splits(const hz_token_attention& a) {
  const int64_t G = a.H / a.Hk, blocks = a.B * a.Hk * ((a.Nk + kBlock - 1) / kBlock);
  int64_t heads = 1;
  while (heads < G && (blocks * heads < 512 || G % heads != 0)) ++heads;
  return {nullptr, a.B * a.Nk * a.Hk * a.D, static_cast<int>(heads) * share_of(blocks * heads, a.Nq, 512), static_cast<int>(heads)};
}

// The two sums are made one after the other in the same memory.
int64_t split_bytes(const hz_token_attention& a) {
  auto bytes = [](const Splits& s, int tensors) { return s.n > 1 ? s.n * tensors * s.elements * static_cast<int64_t>(sizeof(float)) : 0; };
  const int64_t q = bytes(dq_splits(a), 1), kv = bytes(dkv_splits(a), 2);
  return q > kv ? q : kv;
}

int64_t stats_bytes(const hz_token_attention& a) { return a.B * a.Nq * a.H * static_cast<int64_t>(sizeof(RowStats)); }

template <int DP, int PARTS, bool CAP, bool SLOPE>
hipError_t run(const hz_token_attention& a, const hz_token_tensor& dout, void* dq, void* dk, void* dv, void* workspace,
               hipStream_t stream) {
  constexpr int WAVES = PARTS == 1 || DP == 64 ? 8 : 4;
  Params p = make_params(a);
  RowStats* const stats = static_cast<RowStats*>(workspace);
  Splits of_q = dq_splits(a), of_kv = dkv_splits(a);
  of_q.partial = of_kv.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + stats_bytes(a));
  DocTile* const tiles = reinterpret_cast<DocTile*>(static_cast<char*>(workspace) + stats_bytes(a) + split_bytes(a));
  if (hipError_t err = launch_docs(a, p, true, tiles, stream); err != hipSuccess) return err;
  const int64_t nq = a.B * a.H * ((a.Nq + kBlock - 1) / kBlock) * of_q.n, nk = a.B * a.Hk * ((a.Nk + kBlock - 1) / kBlock) * of_kv.n;
  token_dq_kernel<DP, PARTS, CAP, SLOPE><<<static_cast<unsigned>(nq), 256, 0, stream>>>(p, dout, dq, stats, tiles, of_q);
  launch_sum<PARTS>(of_q, 1, dq, nullptr, stream);
  token_dkv_kernel<DP, PARTS, CAP, SLOPE, WAVES><<<static_cast<unsigned>(nk), 64 * WAVES, 0, stream>>>(p, dout, stats, dk, dv, tiles, of_kv);
  launch_sum<PARTS>(of_kv, 2, dk, dv, stream);
  return hipGetLastError();
}

}  // namespace

int64_t token_attention_bwd_workspace(const hz_token_attention& a) {
  return stats_bytes(a) + split_bytes(a) + doc_bytes(a);
}

hipError_t launch_token_attention_bwd(const hz_token_attention& a, const hz_token_tensor& dout, void* dq, void* dk,
                                      void* dv, void* workspace, hipStream_t stream) {
  auto by_score = [&](auto dp, auto parts, auto cap) {
    return a.slopes != nullptr ? run<dp.value, parts.value, cap.value, true>(a, dout, dq, dk, dv, workspace, stream)
                               : run<dp.value, parts.value, cap.value, false>(a, dout, dq, dk, dv, workspace, stream);
  };
  auto by_type = [&](auto dp) {
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 3> Split;
    if (a.dtype == HZ_DTYPE_BF16)
      return a.softcap > 0.f ? by_score(dp, One{}, std::true_type{}) : by_score(dp, One{}, std::false_type{});
    return a.softcap > 0.f ? by_score(dp, Split{}, std::true_type{}) : by_score(dp, Split{}, std::false_type{});
  };
  if (a.D <= 32) return by_type(std::integral_constant<int, 32>{});
  if (a.D <= 64) return by_type(std::integral_constant<int, 64>{});
  return by_type(std::integral_constant<int, 128>{});
}

}  // namespace hz
