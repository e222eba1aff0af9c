// Forward of the token attention (formulas and masks: include/hz_token.h; operand layouts:
// token_device.h).
//
// Two kernels. Many queries: a workgroup of four waves owns 128 queries of a head, 32 a wave, and
// streams the keys they can see through LDS in tiles of KB with the running maximum and sum of the
// softmax; the next tile's loads are in flight during a tile's products. Few queries (at most 32 rows of
// query and head share a key head): a wave owns a run of keys and all of those rows, so the
// cache is read once, and a second kernel joins the runs.
#include "token_device.h"

namespace hz {
namespace {

using namespace token;

constexpr int kThreads = 256;
constexpr int kQB = 128;  // queries a workgroup

// Keys a tile: three parts of 64 keys at 128 elements would leave room for one workgroup a CU.
template <int DP, int PARTS>
constexpr int kKeys = (DP == 128 && PARTS == 3) ? 32 : 64;

// One lane's running softmax of one query, base 2.
struct Running {
  float m = kNegInf, l = 0.f;
};

// Scores of a 32-key block (first key k0) from their dot products, base 2, hidden ones -inf.
// docs: the block's documents in LDS, or null.
template <int PARTS, bool CAP>
__device__ __forceinline__ void scores(v16f& s, const Params& p, const Sight& me, float slope2, int k0, int hh,
                                       bool masked, const int* docs) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x = s[i];
    if constexpr (CAP) x = tanh_of<PARTS>(x * p.to_tanh);
    s[i] = x * p.to_score2;
  }
  if (slope2 != 0.f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] -= slope2 * static_cast<float>(abs(me.pos - (k0 + row_of(i, hh))));
  }
  if (masked) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = k0 + row_of(i, hh) <= me.last ? s[i] : kNegInf;
    if (docs != nullptr) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = docs[row_of(i, hh)] == me.doc ? s[i] : kNegInf;
    }
  }
}

// Softmax weights of NB score blocks against the running maximum; returns the factor of what was
// summed before.
template <int NB>
__device__ __forceinline__ float weigh(v16f (&s)[NB], Running& r) {
  float top = kNegInf;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
  top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
  const float m = fmaxf(r.m, top), base = m == kNegInf ? 0.f : m;  // nothing seen yet: weights of 2^-inf
  const float alpha = fast_exp2(r.m - base);
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[n][i] = fast_exp2(s[n][i] - base);
      sum += s[n][i];
    }
  r.m = m;
  r.l = r.l * alpha + sum;  // this half wave's keys; both halves' at the end
  return alpha;
}

template <int DP, int PARTS, bool CAP>
__global__ void __launch_bounds__(kThreads) token_fwd_kernel(Params p) {
  constexpr int KB = kKeys<DP, PARTS>, NB = KB / 32, DT = DP / 32, CH = DP / 8;
  constexpr int LOADS = KB * CH / kThreads;  // chunks a thread and tensor
  constexpr int STEP = kThreads / CH;        // rows between a thread's chunks
  typedef Tile<KB, DP, PARTS> KV;
  __shared__ __align__(16) uint16_t k_lds[KV::kPlane * PARTS], v_lds[KV::kPlane * PARTS];
  __shared__ int doc_lds[KB];
  const KV kt{k_lds}, vt{v_lds};
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hh = lane >> 5, c = lane & 31;
  const int tiles = (p.Nq + kQB - 1) / kQB;
  int64_t id = xcd_logical_block(blockIdx.x, gridDim.x);
  const int h = static_cast<int>(id % p.H);
  id /= p.H;
  const int q0 = static_cast<int>(tiles - 1 - id % tiles) * kQB;  // the longest rows of a causal mask first
  const int b = static_cast<int>(id / tiles);
  const int hk = h / p.G, n = kv_length(p, b);

  const int i = q0 + 32 * wave + c, row = i < p.Nq ? i : p.Nq - 1;
  const Sight me(p, b, row, n);
  const float slope2 = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
  const int last_row = min(q0 + kQB, p.Nq) - 1;
  const int end = Sight(p, b, last_row, n).last + 1;  // the last query sees the most keys
  const int wave_first = __builtin_amdgcn_readfirstlane(me.last);
  const int wave_last = Sight(p, b, min(q0 + 32 * wave + 31, p.Nq - 1), n).last;

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

  const int lr = tid / CH, lc = tid % CH;
  Raw8<PARTS> rk[LOADS], rv[LOADS];
  int rdoc = -1;
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int key = k0 + lr + STEP * j;
      bool on = key < n && 8 * lc < p.D;
      rk[j].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + 8 * lc, on);
      if (p.documents != nullptr && on) on = key_document(p, b, key) >= 0;  // padding may hold anything
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
    if (k0 > wave_last) continue;  // no query of this wave sees the tile
    v16f s[NB];
    const bool masked = p.documents != nullptr || k0 + KB - 1 > wave_first;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s[nb] = v16f{};
#pragma unroll
      for (int ds = 0; ds < DP / 16; ++ds) s[nb] = mma(kt.rows(32 * nb, ds, lane), q[ds], s[nb]);
      scores<PARTS, CAP>(s[nb], p, me, slope2, k0 + 32 * nb, hh, masked, p.documents != nullptr ? doc_lds + 32 * nb : nullptr);
    }
    const float alpha = weigh<NB>(s, run);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
#pragma unroll
    for (int st = 0; st < 2 * NB; ++st) {
      const Frag<PARTS> w = frag_of<PARTS>(s[st / 2], st % 2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mma(vt.columns(16 * st, dt, lane), w, o[dt]);
    }
  }
  const float l = xor32_pair_sum(run.l);
  if (i >= p.Nq) return;
  const int64_t at = (static_cast<int64_t>(b) * p.Nq + i) * p.H + h;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < p.D)
        store_four<PARTS>(p.out, at * p.D + d, o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv,
                          o[dt][4 * g + 3] * inv);
    }
  if (p.lse != nullptr && hh == 0) p.lse[at] = l == 0.f ? kNegInf : (run.m + log2f(l)) * kLn2;
}

// Few queries: column pr of the products is query pr / G, head hk G + pr % G. Runs of `chunk` keys, one a
// wave; partial [rows of (b, i, h)][runs][D] sums and stats [..][runs][2] (maximum, sum).
template <int DP, int PARTS, bool CAP>
__global__ void __launch_bounds__(kThreads) token_few_kernel(Params p, int chunk, int runs, float* partial, float* stats) {
  constexpr int DT = DP / 32, CH = DP / 8, LOADS = 32 * CH / 64, STEP = 64 / CH;
  typedef Tile<32, DP, PARTS> V;
  __shared__ __align__(16) uint16_t v_lds[4][V::kPlane * PARTS];
  __shared__ int doc_lds[4][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, hh = lane >> 5, c = lane & 31;
  const V vt{v_lds[wave]};
  const int per = (runs + 3) / 4;
  int64_t id = blockIdx.x;
  const int run_id = 4 * static_cast<int>(id % per) + wave;
  id /= per;
  const int hk = static_cast<int>(id % p.Hk), b = static_cast<int>(id / p.Hk);
  const int n = kv_length(p, b), first = run_id * chunk;
  if (run_id >= runs || first >= n) return;  // waves share nothing: no barriers
  const int stop = min(n, first + chunk);
  const int rows = p.Nq * p.G, pr = c < rows ? c : rows - 1, i = pr / p.G, h = hk * p.G + pr % p.G;
  const Sight me(p, b, i, n);
  const float slope2 = p.slopes != nullptr ? p.slopes[h] * kLog2e : 0.f;
  Frag<PARTS> q[DP / 16];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    Raw8<PARTS> r;
    const int d = 16 * s + 8 * hh;
    r.load(p.q.data, b * p.q.batch + i * p.q.token + h * p.q.head + d, d < p.D);
    q[s] = frag(r);
  }
  v16f o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = v16f{};
  Running run;
  const int lr = lane / CH, lc = lane % CH;
  for (int k0 = first; k0 < stop; k0 += 32) {
    Raw8<PARTS> rk[DP / 16], rv[LOADS];
    const int key = k0 + c;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * hh;
      rk[s].load(p.k.data, b * p.k.batch + key * p.k.token + hk * p.k.head + d, key < n && d < p.D);
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int kv = k0 + lr + STEP * j;
      bool on = kv < n && 8 * lc < p.D;
      if (p.documents != nullptr && on) on = key_document(p, b, kv) >= 0;
      rv[j].load(p.v.data, b * p.v.batch + kv * p.v.token + hk * p.v.head + 8 * lc, on);
    }
    if (p.documents != nullptr && lane < 32) doc_lds[wave][lane] = key < n ? key_document(p, b, key) : -1;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) vt.put(lr + STEP * j, lc, frag(rv[j]));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    v16f s[1] = {v16f{}};
#pragma unroll
    for (int ds = 0; ds < DP / 16; ++ds) s[0] = mma(frag(rk[ds]), q[ds], s[0]);
    scores<PARTS, CAP>(s[0], p, me, slope2, k0, hh, true, p.documents != nullptr ? doc_lds[wave] : nullptr);
    const float alpha = weigh<1>(s, run);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const Frag<PARTS> w = frag_of<PARTS>(s[0], st);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mma(vt.columns(16 * st, dt, lane), w, o[dt]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  const float l = xor32_pair_sum(run.l);
  if (c >= rows) return;
  const int64_t at = ((static_cast<int64_t>(b) * p.Nq + i) * p.H + h) * runs + run_id;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * hh;
      if (d < p.D)
        *reinterpret_cast<v4f*>(partial + at * p.D + d) =
            v4f{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
    }
  if (hh == 0) {
    stats[at * 2] = run.m;
    stats[at * 2 + 1] = l;
  }
}

// Joins the runs of one row of (b, i, h): a workgroup of 64 threads a row.
template <int PARTS>
__global__ void __launch_bounds__(64) token_join_kernel(Params p, int chunk, int runs, const float* partial,
                                                        const float* stats) {
  const int64_t at = blockIdx.x;
  const int b = static_cast<int>(at / (static_cast<int64_t>(p.Nq) * p.H)), lane = threadIdx.x;
  const int used = (kv_length(p, b) + chunk - 1) / chunk;
  const float* const st = stats + at * runs * 2;
  float m = kNegInf;
  for (int r = lane; r < used; r += 64) m = fmaxf(m, st[2 * r]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const float base = m == kNegInf ? 0.f : m;
  float l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int r = 0; r < used; ++r) {
    const float a = fast_exp2(st[2 * r] - base);
    l += a * st[2 * r + 1];
    const float* const o = partial + (at * runs + r) * p.D;
    if (2 * lane < p.D) {
      o0 += a * o[2 * lane];
      o1 += a * o[2 * lane + 1];
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  if (2 * lane < p.D) {
    if constexpr (PARTS == 1)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + at * p.D + 2 * lane) = pack2_bf16(o0 * inv, o1 * inv);
    else
      *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at * p.D + 2 * lane) = make_float2(o0 * inv, o1 * inv);
  }
  if (p.lse != nullptr && lane == 0) p.lse[at] = l == 0.f ? kNegInf : (m + log2f(l)) * kLn2;
}

// The few-query kernel takes the calls whose rows of query and head fit the 32 columns of one product.
bool few(const hz_token_attention& a) { return a.Nq * (a.H / a.Hk) <= 32; }

// Keys a run: about 8192 waves in all, at least one block of 32 keys.
int run_keys(const hz_token_attention& a) {
  const int64_t keys = (a.B * a.Hk * a.Nk + 8191) / 8192;
  return static_cast<int>((keys + 31) / 32 * 32);
}
int runs_of(const hz_token_attention& a) {
  const int c = run_keys(a);
  return static_cast<int>((a.Nk + c - 1) / c);
}

template <int DP, int PARTS, bool CAP>
hipError_t run(const hz_token_attention& a, void* workspace, hipStream_t stream) {
  const Params p = make_params(a);
  if (!few(a)) {
    const int64_t grid = a.B * a.H * ((a.Nq + kQB - 1) / kQB);
    token_fwd_kernel<DP, PARTS, CAP><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
    return hipGetLastError();
  }
  const int chunk = run_keys(a), runs = runs_of(a);
  float* const partial = static_cast<float*>(workspace);
  float* const stats = partial + a.B * a.Nq * a.H * runs * a.D;
  token_few_kernel<DP, PARTS, CAP><<<static_cast<unsigned>(a.B * a.Hk * ((runs + 3) / 4)), kThreads, 0, stream>>>(
      p, chunk, runs, partial, stats);
  token_join_kernel<PARTS><<<static_cast<unsigned>(a.B * a.Nq * a.H), 64, 0, stream>>>(p, chunk, runs, partial, stats);
  return hipGetLastError();
}

}  // namespace

int64_t token_attention_fwd_workspace(const hz_token_attention& a) {
  if (!few(a)) return 0;
  return a.B * a.Nq * a.H * runs_of(a) * (a.D + 2) * static_cast<int64_t>(sizeof(float));
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
