// Reverse mode of the token attention (formulas and masks: include/hz_token.h; operand layouts:
// token_device.h).
//
// Two kernels, each with its sums in registers, so that nothing is added atomically: one owns queries and
// streams keys (dq, and rowsum(dout out) for the other), one owns keys and streams the queries of
// every head that shares them (dk, dv). Both rebuild P = exp(s - lse) from the forward's lse: seven products
// a tile pair where one kernel with atomic dq sums would need five.
#include "token_device.h"

namespace hz {
namespace {

using namespace token;

constexpr int kThreads = 256;
constexpr int kBlock = 128;  // queries (dq) or keys (dk, dv) a workgroup, 32 a wave

// Rows of a streamed tile: two tensors, float32 ones in three parts.
template <int DP, int PARTS>
constexpr int kRows = (DP == 128 && PARTS == 3) ? 32 : 64;

// Weight and score gradient (without the scale) of one visible pair, from its dot product x, its dP and the
// distance between query and key.
template <int PARTS, bool CAP>
__device__ __forceinline__ void pair(const Params& p, float x, float dp, float slope2, int distance, float lse2,
                                     float delta, bool seen, float& w, float& ds) {
  float t = 0.f;
  if constexpr (CAP) {
    t = tanh_of<PARTS>(x * p.to_tanh);
    x = t;
  }
  const float s = x * p.to_score2 - slope2 * static_cast<float>(distance);
  w = seen ? fast_exp2(s - lse2) : 0.f;
  float g = w * (dp - delta);
  if constexpr (CAP) g *= 1.f - t * t;
  ds = seen ? g : 0.f;
}

template <int DP, int PARTS, bool CAP>
__global__ void __launch_bounds__(kThreads) token_dq_kernel(Params p, hz_token_tensor dout, void* dq, float* deltas) {
  constexpr int KB = kRows<DP, PARTS>, NB = KB / 32, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = KB * CH / kThreads, STEP = kThreads / CH;
  typedef Tile<KB, DP, PARTS> KV;
  __shared__ __align__(16) uint16_t k_lds[KV::kPlane * PARTS], v_lds[KV::kPlane * PARTS];
  __shared__ int doc_lds[KB];
  const KV kt{k_lds}, vt{v_lds};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  const int tiles = (p.Nq + kBlock - 1) / kBlock;
  int64_t id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int h = static_cast<int>(id % p.H);
  id /= p.H;
  const int q0 = static_cast<int>(tiles - 1 - id % tiles) * kBlock;
  const int b = static_cast<int>(id / tiles);
  const int hk = h / p.G, n = kv_length(p, b);
  const int i = q0 + 32 * wave + c, row = i < p.Nq ? i : p.Nq - 1;
  const Sight me(p, b, row, n);
  const float slope2 = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
  const int end = Sight(p, b, min(q0 + kBlock, p.Nq) - 1, n).last + 1;
  const int wave_first = __builtin_amdgcn_readfirstlane(me.last);
  const int wave_last = Sight(p, b, min(q0 + 32 * wave + 31, p.Nq - 1), n).last;
  const int64_t at = (static_cast<int64_t>(b) * p.Nq + row) * p.H + h;

  Frag<PARTS> q[DP / 16], go[DP / 16];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> rq, rg, ro;
    const int d = 16 * s + 8 * hh;
    rq.load(p.q.data, b * p.q.batch + row * p.q.token + h * p.q.head + d, d < p.D);
    rg.load(dout.data, b * dout.batch + row * dout.token + h * dout.head + d, d < p.D);
    ro.load(p.out, at * p.D + d, d < p.D);
    float x[8], y[8];
    floats(rg, x);
    floats(ro, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += x[j] * y[j];
    q[s] = frag(rq);
    go[s] = frag(rg);
  }
  delta = xor32_pair_sum(delta);
  if (i < p.Nq && hh == 0) deltas[at] = delta;
  float lse2 = p.lse[at] * kLog2e;
  if (lse2 == kNegInf) lse2 = 0.f;  // a row that sees nothing
  v16f acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = v16f{};

  const int lr = tid / CH, lc = tid % CH;
  Raw8<PARTS> rk[LOADS], rv[LOADS];
  int rdoc = -1;
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int key = k0 + lr + STEP * j;
      bool on = key < n && 8 * lc < p.D;
      if (p.documents != nullptr && on) on = key_document(p, b, key) >= 0;  // padding may hold anything
      rk[j].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + 8 * lc, on);
      rv[j].load(p.v.data, b * p.v.batch + key * p.v.token + hk * p.v.head + 8 * lc, on);
    }
    if (p.documents != nullptr && tid < KB) rdoc = k0 + tid < n ? key_document(p, b, k0 + tid) : -1;
  };
  if (end > 0) load(0);
  for (int k0 = 0; k0 < end; k0 += KB) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      kt.put(lr + STEP * j, lc, frag(rk[j]));
      vt.put(lr + STEP * j, lc, frag(rv[j]));
    }
    if (p.documents != nullptr && tid < KB) doc_lds[tid] = rdoc;
    __syncthreads();
    if (k0 + KB < end) load(k0 + KB);
    if (k0 > wave_last) continue;
    const bool masked = p.documents != nullptr || k0 + KB - 1 > wave_first;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      v16f s = v16f{}, dp = v16f{};
#pragma unroll
      for (int ds = 0; ds < DP / 16; ++ds) {
        s = mma(kt.rows(32 * nb, ds, lane), q[ds], s);
        dp = mma(vt.rows(32 * nb, ds, lane), go[ds], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = 32 * nb + row_of(e, hh), key = k0 + r;
        bool seen = true;
        if (masked) {
          seen = key <= me.last;
          if (p.documents != nullptr) seen = seen && doc_lds[r] == me.doc;
        }
        float w, g;
        pair<PARTS, CAP>(p, s[e], dp[e], slope2, abs(me.pos - key), lse2, delta, seen, w, g);
        s[e] = g;
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const Frag<PARTS> g = frag_of<PARTS>(s, st);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mma(kt.columns(32 * nb + 16 * st, dt, lane), g, acc[dt]);
      }
    }
  }
  if (i >= p.Nq) return;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < p.D)
        store_four<PARTS>(dq, at * p.D + d, acc[dt][4 * g] * p.scale, acc[dt][4 * g + 1] * p.scale,
                          acc[dt][4 * g + 2] * p.scale, acc[dt][4 * g + 3] * p.scale);
    }
}

template <int DP, int PARTS, bool CAP>
__global__ void __launch_bounds__(kThreads) token_dkv_kernel(Params p, hz_token_tensor dout, const float* deltas, void* dk,
                                                             void* dv) {
  constexpr int QB = kRows<DP, PARTS>, NB = QB / 32, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = QB * CH / kThreads, STEP = kThreads / CH;
  typedef Tile<QB, DP, PARTS> QT;
  __shared__ __align__(16) uint16_t q_lds[QT::kPlane * PARTS], g_lds[QT::kPlane * PARTS];
  __shared__ __align__(16) float lse_lds[QB], delta_lds[QB];
  __shared__ __align__(16) int last_lds[QB], doc_lds[QB];
  const QT qt{q_lds}, gt{g_lds};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  const int tiles = (p.Nk + kBlock - 1) / kBlock;
  int64_t id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int hk = static_cast<int>(id % p.Hk);
  id /= p.Hk;
  const int key0 = static_cast<int>(id % tiles) * kBlock;  // the first keys are seen by the most queries
  const int b = static_cast<int>(id / tiles);
  const int n = kv_length(p, b);
  const int wave0 = key0 + 32 * wave, key = wave0 + c, row = key < n ? key : max(n - 1, 0);
  const int my_doc = p.documents != nullptr && key < n ? key_document(p, b, key) : -1;

  Frag<PARTS> k[DP / 16], v[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> rk, rv;
    const int d = 16 * s + 8 * hh;
    rk.load(p.k.data, b * p.k.batch + row * p.k.token + hk * p.k.head + d, key < n && d < p.D);
    rv.load(p.v.data, b * p.v.batch + row * p.v.token + hk * p.v.head + d, key < n && d < p.D);
    k[s] = frag(rk);
    v[s] = frag(rv);
  }
  v16f ak[DT], av[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ak[dt] = v16f{}, av[dt] = v16f{};

  // the first query that may see a key of this block
  int begin = 0;
  if (p.causal && key0 >= (p.prefix != nullptr ? p.prefix[b] : 0)) begin = max(0, key0 - (n - p.Nq));
  begin = key0 < n ? begin / QB * QB : p.Nq;
  const int lr = tid / CH, lc = tid % CH;
  Raw8<PARTS> rq[LOADS], rg[LOADS];
  float rlse = 0.f, rdelta = 0.f;
  int rlast = -1, rdoc = kNoDocument;
  auto load = [&](int h, int q0) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = q0 + lr + STEP * j;
      bool on = i < p.Nq && 8 * lc < p.D;
      if (on) on = p.lse[(static_cast<int64_t>(b) * p.Nq + i) * p.H + h] != kNegInf;  // padding may hold anything
      rq[j].load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + 8 * lc, on);
      rg[j].load(dout.data, b * dout.batch + i * dout.token + h * dout.head + 8 * lc, on);
    }
    if (tid < QB) {
      const int i = q0 + tid;
      rlse = 0.f, rdelta = 0.f, rlast = -1, rdoc = kNoDocument;
      if (i < p.Nq) {
        const int64_t at = (static_cast<int64_t>(b) * p.Nq + i) * p.H + h;
        rlse = p.lse[at] * kLog2e;
        if (rlse == kNegInf) rlse = 0.f;
        rdelta = deltas[at];
        const Sight s(p, b, i, n);
        rlast = s.last;
        rdoc = s.doc;
      }
    }
  };
  for (int g = 0; g < p.G; ++g) {
    const int h = hk * p.G + g;
    const float slope2 = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
    if (begin < p.Nq) load(h, begin);
    for (int q0 = begin; q0 < p.Nq; q0 += QB) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        qt.put(lr + STEP * j, lc, frag(rq[j]));
        gt.put(lr + STEP * j, lc, frag(rg[j]));
      }
      if (tid < QB) lse_lds[tid] = rlse, delta_lds[tid] = rdelta, last_lds[tid] = rlast, doc_lds[tid] = rdoc;
      __syncthreads();
      if (q0 + QB < p.Nq) load(h, q0 + QB);
      const int top = min(q0 + QB, p.Nq) - 1 - q0;
      if (last_lds[top] < wave0) continue;  // no query of the tile sees a key of this wave
      const bool masked = p.documents != nullptr || q0 + QB > p.Nq || last_lds[0] < wave0 + 31;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        v16f s = v16f{}, dp = v16f{};
#pragma unroll
        for (int ds = 0; ds < DP / 16; ++ds) {
          s = mma(qt.rows(32 * nb, ds, lane), k[ds], s);
          dp = mma(gt.rows(32 * nb, ds, lane), v[ds], dp);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int r = 32 * nb + row_of(e, hh);
          bool seen = true;
          if (masked) {
            seen = key <= last_lds[r];
            if (p.documents != nullptr) seen = seen && doc_lds[r] == my_doc;
          }
          float w, gs;
          pair<PARTS, CAP>(p, s[e], dp[e], slope2, abs(n - p.Nq + q0 + r - key), lse_lds[r], delta_lds[r], seen, w, gs);
          s[e] = w;
          dp[e] = gs;
        }
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Frag<PARTS> w = frag_of<PARTS>(s, st), gs = frag_of<PARTS>(dp, st);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            av[dt] = mma(gt.columns(32 * nb + 16 * st, dt, lane), w, av[dt]);
            ak[dt] = mma(qt.columns(32 * nb + 16 * st, dt, lane), gs, ak[dt]);
          }
        }
      }
    }
  }
  if (key >= p.Nk) return;
  const int64_t at = ((static_cast<int64_t>(b) * p.Nk + key) * p.Hk + hk) * p.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < p.D) {
        store_four<PARTS>(dk, at + d, ak[dt][4 * g] * p.scale, ak[dt][4 * g + 1] * p.scale, ak[dt][4 * g + 2] * p.scale,
                          ak[dt][4 * g + 3] * p.scale);
        store_four<PARTS>(dv, at + d, av[dt][4 * g], av[dt][4 * g + 1], av[dt][4 * g + 2], av[dt][4 * g + 3]);
      }
    }
}

template <int DP, int PARTS, bool CAP>
hipError_t run(const hz_token_attention& a, const hz_token_tensor& dout, void* dq, void* dk, void* dv, void* workspace,
               hipStream_t stream) {
  const Params p = make_params(a);
  float* const deltas = static_cast<float*>(workspace);
  const int64_t nq = a.B * a.H * ((a.Nq + kBlock - 1) / kBlock), nk = a.B * a.Hk * ((a.Nk + kBlock - 1) / kBlock);
  token_dq_kernel<DP, PARTS, CAP><<<static_cast<unsigned>(nq), kThreads, 0, stream>>>(p, dout, dq, deltas);
  token_dkv_kernel<DP, PARTS, CAP><<<static_cast<unsigned>(nk), kThreads, 0, stream>>>(p, dout, deltas, dk, dv);
  return hipGetLastError();
}

}  // namespace

int64_t token_attention_bwd_workspace(const hz_token_attention& a) {
  return a.B * a.Nq * a.H * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_token_attention_bwd(const hz_token_attention& a, const hz_token_tensor& dout, void* dq, void* dk,
                                      void* dv, void* workspace, hipStream_t stream) {
  auto by_type = [&](auto dp) {
    constexpr int DP = dp.value;
    if (a.dtype == HZ_DTYPE_BF16)
      return a.softcap > 0.f ? run<DP, 1, true>(a, dout, dq, dk, dv, workspace, stream)
                             : run<DP, 1, false>(a, dout, dq, dk, dv, workspace, stream);
    return a.softcap > 0.f ? run<DP, 3, true>(a, dout, dq, dk, dv, workspace, stream)
                           : run<DP, 3, false>(a, dout, dq, dk, dv, workspace, stream);
  };
  if (a.D <= 32) return by_type(std::integral_constant<int, 32>{});
  if (a.D <= 64) return by_type(std::integral_constant<int, 64>{});
  return by_type(std::integral_constant<int, 128>{});
}

}  // namespace hz
