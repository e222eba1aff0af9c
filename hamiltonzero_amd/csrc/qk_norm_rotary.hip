// Norms of queries and keys for each head with the position rotation in the same pass, and their
// reverse mode (formulas: include/hz_token.h).
//
// One head of D elements is held by L = D / 8 lanes, eight elements a lane as two chunks of four,
// chosen so that both elements of each rotated pair are in one lane and no lane exchanges data but
// for the sum of squares: with half-split pairs lane t holds elements 4 t .. 4 t + 3 and
// n_freqs + 4 t .. + 3, with interleaved ones (and behind the rotated part) 8 t .. 8 t + 7. Either
// way it turns pairs 4 t .. 4 t + 3, so a lane's four angles serve every head of a token: they are
// formed once a token, in float64 turns (an angle at position 10^5 has no bits to lose in float32's
// 24), and the workgroup's lanes then loop over the token's query and key heads.
// Bound by the bytes: x is read and y written once; the backward reads x and dy and writes dx.
#include "mhsea_device.h"
#include "token_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 2048;  // of the backward: rows of partial weight gradients

struct NormParams {
  hz_token_tensor q, k, qo, ko;
  const float *wq, *wk;
  const double* freqs;
  const int32_t* positions;
  int64_t tokens;
  int N, H, HT, D, nf, interleaved;
  float eps;
};

// Where a lane's two chunks of four elements lie in its head, and its four angles.
struct Lane {
  int o0, o1;
  bool on, turns;
  __device__ __forceinline__ Lane(const NormParams& p, int t) {
    on = 8 * t < p.D;
    turns = 4 * t < p.nf;
    const bool split = turns && !p.interleaved;
    o0 = split ? 4 * t : 8 * t;
    o1 = split ? p.nf + 4 * t : 8 * t + 4;
  }
};

__device__ __forceinline__ void angles(const NormParams& p, int64_t token, int t, float (&cs)[4], float (&sn)[4]) {
  const double pos = p.positions != nullptr ? p.positions[token] : static_cast<int>(token % p.N);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double turn = pos * p.freqs[4 * t + i] * 0.15915494309189533577;  // radians to turns
    turn -= rint(turn);
    sincospif(2.f * static_cast<float>(turn), &sn[i], &cs[i]);
  }
}

// The eight elements turned by their four angles (dir 1) or back (dir -1).
__device__ __forceinline__ void turn8(float (&x)[8], const float (&cs)[4], const float (&sn)[4], int interleaved,
                                      float dir) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = dir * sn[i];
    if (interleaved) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * cs[i] - b * s;
      x[2 * i + 1] = b * cs[i] + a * s;
    } else {
      const float a = x[i], b = x[i + 4];
      x[i] = a * cs[i] - b * s;
      x[i + 4] = b * cs[i] + a * s;
    }
  }
}

template <int GS>
__device__ __forceinline__ float head_sum(float x) {
#pragma unroll
  for (int m = 1; m < GS; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}

template <class S>
__device__ __forceinline__ void load8(const void* base, int64_t off, const Lane& l, float (&x)[8]) {
  const float4 a = load4<S>(base, off + l.o0), b = load4<S>(base, off + l.o1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <class S>
__device__ __forceinline__ void store8(void* base, int64_t off, const Lane& l, const float (&x)[8]) {
  store4<S>(base, off + l.o0, x[0], x[1], x[2], x[3]);
  store4<S>(base, off + l.o1, x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ void weights(const float* w, const Lane& l, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = w != nullptr && l.on ? w[l.o0 + i] : 1.f;
    x[4 + i] = w != nullptr && l.on ? w[l.o1 + i] : 1.f;
  }
}

// A workgroup's slots of GS lanes: all on one token's heads, or on several tokens where their heads
// are few.
struct Slots {
  int per, token, head, step;  // tokens a workgroup; this slot's token and first head; heads a step
  bool on;
  __device__ __forceinline__ Slots(int HT, int gs) {
    const int n = kThreads / gs, s = threadIdx.x / gs;
    per = n / HT > 1 ? n / HT : 1;
    token = per > 1 ? s / HT : 0;
    head = per > 1 ? s % HT : s;
    step = per > 1 ? HT : n;
    on = token < per;
  }
};

__device__ __forceinline__ int64_t head_offset(const hz_token_tensor& x, int64_t b, int64_t n, int h) {
  return b * x.batch + n * x.token + h * x.head;
}

template <class S, int GS>
__global__ void __launch_bounds__(kThreads) norm_rotary_fwd_kernel(NormParams p) {
  const int t = threadIdx.x % GS;
  const Lane lane(p, t);
  const Slots slot(p.HT, GS);
  float wq[8], wk[8];
  weights(p.wq, lane, wq);
  weights(p.wk, lane, wk);
  if (!slot.on) return;
  for (int64_t tok = static_cast<int64_t>(blockIdx.x) * slot.per + slot.token; tok < p.tokens;
       tok += static_cast<int64_t>(gridDim.x) * slot.per) {
    const int64_t b = tok / p.N, n = tok - b * p.N;
    float cs[4], sn[4];
    if (lane.turns) angles(p, tok, t, cs, sn);
    for (int h = slot.head; h < p.HT; h += slot.step) {
      const bool is_q = h < p.H;
      const hz_token_tensor& in = is_q ? p.q : p.k;
      const hz_token_tensor& out = is_q ? p.qo : p.ko;
      const int hd = is_q ? h : h - p.H;
      float x[8] = {};
      if (lane.on) load8<S>(in.data, head_offset(in, b, n, hd), lane, x);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      const float r = 1.f / sqrtf(head_sum<GS>(ss) / static_cast<float>(p.D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= r * (is_q ? wq[i] : wk[i]);
      if (lane.turns) turn8(x, cs, sn, p.interleaved, 1.f);
      if (lane.on) store8<S>(out.data, head_offset(out, b, n, hd), lane, x);
    }
  }
}

// q and k: the forward's inputs; qo and ko: the cotangents. partial: [gridDim.x][2][D].
template <class S, int GS>
__global__ void __launch_bounds__(kThreads) norm_rotary_bwd_kernel(NormParams p, void* dq, void* dk, float* partial) {
  __shared__ float red[kThreads * 8];
  const int t = threadIdx.x % GS;
  const Lane lane(p, t);
  const Slots slot(p.HT, GS);
  float wq[8], wk[8], aq[8] = {}, ak[8] = {};
  weights(p.wq, lane, wq);
  weights(p.wk, lane, wk);
  const int Hk = p.HT - p.H;
  for (int64_t tok = static_cast<int64_t>(blockIdx.x) * slot.per + slot.token; slot.on && tok < p.tokens;
       tok += static_cast<int64_t>(gridDim.x) * slot.per) {
    const int64_t b = tok / p.N, n = tok - b * p.N;
    float cs[4], sn[4];
    if (lane.turns) angles(p, tok, t, cs, sn);
    for (int h = slot.head; h < p.HT; h += slot.step) {
      const bool is_q = h < p.H;
      const hz_token_tensor& in = is_q ? p.q : p.k;
      const hz_token_tensor& cot = is_q ? p.qo : p.ko;
      const int hd = is_q ? h : h - p.H;
      float x[8] = {}, g[8] = {};
      if (lane.on) {
        load8<S>(in.data, head_offset(in, b, n, hd), lane, x);
        load8<S>(cot.data, head_offset(cot, b, n, hd), lane, g);
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
      const float r = 1.f / sqrtf(head_sum<GS>(ss) / static_cast<float>(p.D) + p.eps);
      if (lane.turns) turn8(g, cs, sn, p.interleaved, -1.f);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= r;
        const float gx = g[i] * x[i];
        aq[i] += is_q ? gx : 0.f;
        ak[i] += is_q ? 0.f : gx;
        g[i] *= is_q ? wq[i] : wk[i];
        dot += g[i] * x[i];
      }
      dot = head_sum<GS>(dot) / static_cast<float>(p.D);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = r * (g[i] - x[i] * dot);
      if (lane.on)
        store8<S>(is_q ? dq : dk, (tok * (is_q ? p.H : Hk) + hd) * p.D, lane, x);
    }
  }
  // the workgroup's weight gradients: one row of slots after the other, so their order is fixed
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[i * kThreads + threadIdx.x] = which == 0 ? aq[i] : ak[i];
    __syncthreads();
    for (int d = threadIdx.x; d < GS * 8; d += kThreads) {
      const int tt = d / 8, i = d % 8;
      const Lane l(p, tt);
      if (!l.on) continue;
      float sum = 0.f;
      for (int s = 0; s < kThreads / GS; ++s) sum += red[i * kThreads + s * GS + tt];
      partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.D + (i < 4 ? l.o0 + i : l.o1 + i - 4)] = sum;
    }
  }
}

// Column sums of partial [rows][2 D]: 16 columns a workgroup, 64 threads a column.
__global__ void __launch_bounds__(1024) weight_sum_kernel(const float* partial, int rows, int D, float* dw_q,
                                                          float* dw_k) {
  __shared__ float red[64][16];
  const int c = threadIdx.x % 16, r0 = threadIdx.x / 16, col = blockIdx.x * 16 + c;
  float sum = 0.f;
  if (col < 2 * D)
    for (int r = r0; r < rows; r += 64) sum += partial[static_cast<int64_t>(r) * 2 * D + col];
  red[r0][c] = sum;
  __syncthreads();
  for (int m = 32; m > 0; m >>= 1) {
    if (r0 < m) red[r0][c] += red[r0 + m][c];
    __syncthreads();
  }
  if (r0 == 0 && col < 2 * D) {
    float* const dw = col < D ? dw_q : dw_k;
    if (dw != nullptr) dw[col < D ? col : col - D] = red[0][c];
  }
}

NormParams params(const hz_qk_norm_rotary& a) {
  NormParams p{};
  p.q = a.q, p.k = a.k, p.qo = a.q_out, p.ko = a.k_out;
  p.wq = a.w_q, p.wk = a.w_k, p.freqs = a.freqs, p.positions = a.positions;
  p.tokens = a.B * a.N;
  p.N = static_cast<int>(a.N), p.H = static_cast<int>(a.H), p.HT = static_cast<int>(a.H + a.Hk);
  p.D = static_cast<int>(a.D), p.nf = static_cast<int>(a.n_freqs), p.interleaved = a.interleaved;
  p.eps = a.eps;
  return p;
}

int group_size(int64_t D) {
  int gs = 1;
  while (gs * 8 < D) gs *= 2;
  return gs;
}

int64_t blocks(const NormParams& p, int64_t most) {
  const int slots = kThreads / group_size(p.D), per = slots / p.HT > 1 ? slots / p.HT : 1;
  const int64_t n = (p.tokens + per - 1) / per;
  return n < most ? n : most;
}

template <class F>
void by_group(int gs, F f) {
  switch (gs) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    case 16: f(std::integral_constant<int, 16>{}); break;
    default: f(std::integral_constant<int, 32>{}); break;
  }
}

}  // namespace

int64_t qk_norm_rotary_workspace(int64_t tokens, int64_t D) {
  return (tokens < kMaxBlocks ? tokens : kMaxBlocks) * 2 * D * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_qk_norm_rotary_fwd(const hz_qk_norm_rotary& a, hipStream_t stream) {
  const NormParams p = params(a);
  const dim3 grid(static_cast<unsigned>(blocks(p, 1 << 20)));
  by_group(group_size(p.D), [&](auto gs) {
    if (a.dtype == HZ_DTYPE_BF16)
      norm_rotary_fwd_kernel<BF16, gs.value><<<grid, kThreads, 0, stream>>>(p);
    else
      norm_rotary_fwd_kernel<F32, gs.value><<<grid, kThreads, 0, stream>>>(p);
  });
  return hipGetLastError();
}

hipError_t launch_qk_norm_rotary_bwd(const hz_qk_norm_rotary& a, void* dq, void* dk, float* dw_q, float* dw_k,
                                     void* workspace, hipStream_t stream) {
  const NormParams p = params(a);
  const int rows = static_cast<int>(blocks(p, kMaxBlocks));
  float* const partial = static_cast<float*>(workspace);
  by_group(group_size(p.D), [&](auto gs) {
    if (a.dtype == HZ_DTYPE_BF16)
      norm_rotary_bwd_kernel<BF16, gs.value><<<rows, kThreads, 0, stream>>>(p, dq, dk, partial);
    else
      norm_rotary_bwd_kernel<F32, gs.value><<<rows, kThreads, 0, stream>>>(p, dq, dk, partial);
  });
  if (dw_q != nullptr || dw_k != nullptr)
    weight_sum_kernel<<<(2 * p.D + 15) / 16, 1024, 0, stream>>>(partial, rows, p.D, dw_q, dw_k);
  return hipGetLastError();
}

}  // namespace hz
