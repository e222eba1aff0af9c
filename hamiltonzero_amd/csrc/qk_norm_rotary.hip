// Norms of queries and keys for each head with the position rotation in the same pass, and their
// reverse mode (formulas: include/hz_token.h).
//
// One head of D elements is held by L = D / 8 lanes, eight elements a lane as two chunks of four,
// chosen so that both elements of each rotated pair are in one lane and no lane exchanges data but
// for the sum of squares: with half-split pairs lane t holds elements 4 t .. 4 t + 3 and
// n_freqs + 4 t .. + 3, with interleaved ones (and behind the rotated part) 8 t .. 8 t + 7. Either
// way it turns pairs 4 t .. 4 t + 3. A workgroup takes up to four tokens at a time: it forms their angles
// once, in float64 turns (an angle at position 10^5 has no bits to lose in float32's 24), puts the sines
// and cosines into LDS, and then runs over the tokens' query and key heads, the next one's data in flight
// while one is normalised.
// x is read and y written once; the backward reads x and dy and writes dx. float32: bound by those bytes (256 x 225 tokens of 16
// heads of 64: 107 to 116 us, 151 in reverse mode, 4.8 TB/s); bfloat16: by vector instructions beside them, issued 98% of the time (4 x
// 4096 tokens of 40 heads of 128: 90 us, 3.7 TB/s, and 119 us, 4.2 TB/s).
#include "mhsea_device.h"
#include "token_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;     // a workgroup at a time
constexpr int kMaxBlocks = 1024;  // of the backward: rows of partial weight gradients

struct NormParams {
  hz_token_tensor q, k, qo, ko;
  const float *wq, *wk;
  const double* freqs;
  const int32_t* positions;
  int64_t tokens;
  int N, H, HT, D, nf, interleaved, each;  // each: tokens a workgroup at a time
  float eps;
};

// Where a lane's two chunks of four elements lie in its head, and whether they turn.
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

typedef float2 Angles[kMaxTokens][HZ_ROTARY_MAX_HEAD / 2];

__device__ __forceinline__ void put_angles(const NormParams& p, int64_t token0, int count, Angles& angles) {
  for (int a = threadIdx.x; a < count * p.nf; a += kThreads) {
    const int x = a / p.nf, f = a - x * p.nf;
    const int64_t token = token0 + x;
    const double pos = p.positions != nullptr ? p.positions[token] : static_cast<int>(token % p.N);
    double turn = pos * p.freqs[f] * 0.15915494309189533577;  // radians to turns
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * static_cast<float>(turn), &s, &c);
    angles[x][f] = make_float2(c, s);
  }
}

// The eight elements turned by their four angles (dir 1) or back (dir -1). (A template: chosen at run time, the
// pairs' places become indices into an array in scratch memory.)
template <bool INTERLEAVED>
__device__ __forceinline__ void turn8(float (&x)[8], const float2* angle, float dir) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = angle[i].x, s = dir * angle[i].y;
    if constexpr (INTERLEAVED) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * c - b * s;
      x[2 * i + 1] = b * c + a * s;
    } else {
      const float a = x[i], b = x[i + 4];
      x[i] = a * c - b * s;
      x[i + 4] = b * c + a * s;
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
struct Raw {
  Raw4<S> a, b;
  __device__ __forceinline__ void load(const void* base, int64_t off, const Lane& l) {
    a = Raw4<S>::load(base, off + l.o0);
    b = Raw4<S>::load(base, off + l.o1);
  }
  __device__ __forceinline__ void get(float (&x)[8], bool on) const {
    const float4 u = a.f(), v = b.f();
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = on ? x[i] : 0.f;
  }
};

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

// One (token, head) of the tokens at hand: which tensor, and where its head lies in the strided ones and in
// a contiguous one.
struct Item {
  bool is_q;
  int token, head;
  int64_t b, n;
  __device__ __forceinline__ Item(const NormParams& p, int64_t token0, int i) {
    token = i / p.HT;
    const int h = i - token * p.HT;
    is_q = h < p.H;
    head = is_q ? h : h - p.H;
    const int64_t at = token0 + token;
    b = at / p.N;
    n = at - b * p.N;
  }
  // (by value: a reference to one of two kernel arguments would put both into scratch memory)
  __device__ __forceinline__ const void* data(const hz_token_tensor& q, const hz_token_tensor& k) const {
    return is_q ? q.data : k.data;
  }
  __device__ __forceinline__ int64_t offset(const hz_token_tensor& q, const hz_token_tensor& k) const {
    return b * (is_q ? q.batch : k.batch) + n * (is_q ? q.token : k.token) + head * (is_q ? q.head : k.head);
  }
};

template <class S, int GS, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) norm_rotary_fwd_kernel(NormParams p) {
  __shared__ Angles angles;
  constexpr int SLOTS = kThreads / GS;
  const int t = threadIdx.x % GS, slot = threadIdx.x / GS;
  const Lane lane(p, t);
  float wq[8], wk[8];
  weights(p.wq, lane, wq);
  weights(p.wk, lane, wk);
  for (int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.each; token0 < p.tokens;
       token0 += static_cast<int64_t>(gridDim.x) * p.each) {
    const int count = static_cast<int>(p.tokens - token0 < p.each ? p.tokens - token0 : p.each), items = count * p.HT;
    Raw<S> next;
    auto load = [&](int i) {
      if (i < items && lane.on) {
        const Item it(p, token0, i);
        next.load(it.data(p.q, p.k), it.offset(p.q, p.k), lane);
      }
    };
    load(slot);
    put_angles(p, token0, count, angles);
    __syncthreads();
    for (int i = slot; i < items; i += SLOTS) {
      const Item it(p, token0, i);
      float x[8];
      next.get(x, lane.on);
      load(i + SLOTS);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
      const float r = 1.f / sqrtf(head_sum<GS>(ss) / static_cast<float>(p.D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * (it.is_q ? wq[e] : wk[e]);
      if (lane.turns) turn8<INTERLEAVED>(x, &angles[it.token][4 * t], 1.f);
      if (lane.on) store8<S>(const_cast<void*>(it.data(p.qo, p.ko)), it.offset(p.qo, p.ko), lane, x);
    }
    __syncthreads();
  }
}

// q and k: the forward's inputs; qo and ko: the cotangents. partial: [gridDim.x][2][D].
template <class S, int GS, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) norm_rotary_bwd_kernel(NormParams p, void* dq, void* dk, float* partial) {
  __shared__ Angles angles;
  __shared__ float red[kThreads * 8];
  constexpr int SLOTS = kThreads / GS;
  const int t = threadIdx.x % GS, slot = threadIdx.x / GS;
  const Lane lane(p, t);
  float wq[8], wk[8], aq[8] = {}, ak[8] = {};
  weights(p.wq, lane, wq);
  weights(p.wk, lane, wk);
  const int Hk = p.HT - p.H;
  for (int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.each; token0 < p.tokens;
       token0 += static_cast<int64_t>(gridDim.x) * p.each) {
    const int count = static_cast<int>(p.tokens - token0 < p.each ? p.tokens - token0 : p.each), items = count * p.HT;
    Raw<S> next_x, next_g;
    auto load = [&](int i) {
      if (i < items && lane.on) {
        const Item it(p, token0, i);
        next_x.load(it.data(p.q, p.k), it.offset(p.q, p.k), lane);
        next_g.load(it.data(p.qo, p.ko), it.offset(p.qo, p.ko), lane);
      }
    };
    load(slot);
    put_angles(p, token0, count, angles);
    __syncthreads();
    for (int i = slot; i < items; i += SLOTS) {
      const Item it(p, token0, i);
      float x[8], g[8];
      next_x.get(x, lane.on);
      next_g.get(g, lane.on);
      load(i + SLOTS);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
      const float r = 1.f / sqrtf(head_sum<GS>(ss) / static_cast<float>(p.D) + p.eps);
      if (lane.turns) turn8<INTERLEAVED>(g, &angles[it.token][4 * t], -1.f);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= r;
        const float gx = g[e] * x[e];
        aq[e] += it.is_q ? gx : 0.f;
        ak[e] += it.is_q ? 0.f : gx;
        g[e] *= it.is_q ? wq[e] : wk[e];
        dot += g[e] * x[e];
      }
      dot = head_sum<GS>(dot) / static_cast<float>(p.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = r * (g[e] - x[e] * dot);
      if (lane.on)
        store8<S>(it.is_q ? dq : dk, ((token0 + it.token) * (it.is_q ? p.H : Hk) + it.head) * p.D, lane, x);
    }
    __syncthreads();
  }
  // the workgroup's weight gradients: one slot after the other, so their order is fixed
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) red[e * kThreads + threadIdx.x] = which == 0 ? aq[e] : ak[e];
    __syncthreads();
    for (int d = threadIdx.x; d < GS * 8; d += kThreads) {
      const int tt = d / 8, e = d % 8;
      const Lane l(p, tt);
      if (!l.on) continue;
      float sum = 0.f;
#pragma unroll 8
      for (int s = 0; s < SLOTS; ++s) sum += red[e * kThreads + s * GS + tt];
      partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.D + (e < 4 ? l.o0 + e : l.o1 + e - 4)] = sum;
    }
  }
}

// Column sums of partial [rows][2 D]: 4 columns a workgroup, 64 threads a column.
__global__ void __launch_bounds__(kThreads) weight_sum_kernel(const float* partial, int rows, int D, float* dw_q,
                                                              float* dw_k) {
  __shared__ float red[64][4];
  const int c = threadIdx.x % 4, r0 = threadIdx.x / 4, col = blockIdx.x * 4 + c;
  float sum = 0.f;
#pragma unroll 8
  for (int r = r0; r < rows; r += 64) sum += partial[static_cast<int64_t>(r) * 2 * D + col];
  red[r0][c] = sum;
  __syncthreads();
  for (int m = 32; m > 0; m >>= 1) {
    if (r0 < m) red[r0][c] += red[r0 + m][c];
    __syncthreads();
  }
  if (r0 == 0) {
    float* const dw = col < D ? dw_q : dw_k;
    if (dw != nullptr) dw[col < D ? col : col - D] = red[0][c];
  }
}

// Tokens a workgroup at a time: several where that leaves at least `blocks` workgroups, so that the angles are
// formed by all lanes and the loads of several heads overlap (the forwards of
// qk_train_bf16 and qk_train_sites_f32: 90 and 93 us, 115 and 220 with one token).
int tokens_each(int64_t tokens, int64_t blocks) {
  const int64_t n = tokens / blocks;
  return static_cast<int>(n < 1 ? 1 : n > kMaxTokens ? kMaxTokens : n);
}

NormParams params(const hz_qk_norm_rotary& a) {
  NormParams p{};
  p.q = a.q, p.k = a.k, p.qo = a.q_out, p.ko = a.k_out;
  p.wq = a.w_q, p.wk = a.w_k, p.freqs = a.freqs, p.positions = a.positions;
  p.tokens = a.B * a.N;
  p.N = static_cast<int>(a.N), p.H = static_cast<int>(a.H), p.HT = static_cast<int>(a.H + a.Hk);
  p.D = static_cast<int>(a.D), p.nf = static_cast<int>(a.n_freqs), p.interleaved = a.interleaved;
  p.each = tokens_each(p.tokens, kMaxBlocks);
  p.eps = a.eps;
  return p;
}

int64_t blocks(const NormParams& p, int64_t most) {
  const int64_t n = (p.tokens + p.each - 1) / p.each;
  return n < most ? n : most;
}

template <class F>
void by_group(int64_t D, F f) {
  if (D <= 8) return f(std::integral_constant<int, 1>{});
  if (D <= 16) return f(std::integral_constant<int, 2>{});
  if (D <= 32) return f(std::integral_constant<int, 4>{});
  if (D <= 64) return f(std::integral_constant<int, 8>{});
  if (D <= 128) return f(std::integral_constant<int, 16>{});
  f(std::integral_constant<int, 32>{});
}

template <class F>
void by_variant(const hz_qk_norm_rotary& a, F f) {
  by_group(a.D, [&](auto gs) {
    if (a.dtype == HZ_DTYPE_BF16)
      a.interleaved ? f(BF16{}, gs, std::true_type{}) : f(BF16{}, gs, std::false_type{});
    else
      a.interleaved ? f(F32{}, gs, std::true_type{}) : f(F32{}, gs, std::false_type{});
  });
}

}  // namespace

int64_t qk_norm_rotary_workspace(int64_t tokens, int64_t D) {
  return (tokens < kMaxBlocks ? tokens : kMaxBlocks) * 2 * D * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_qk_norm_rotary_fwd(const hz_qk_norm_rotary& a, hipStream_t stream) {
  const NormParams p = params(a);
  const dim3 grid(static_cast<unsigned>(blocks(p, 1 << 20)));
  by_variant(a, [&](auto type, auto gs, auto inter) {
    norm_rotary_fwd_kernel<decltype(type), gs.value, inter.value><<<grid, kThreads, 0, stream>>>(p);
  });
  return hipGetLastError();
}

hipError_t launch_qk_norm_rotary_bwd(const hz_qk_norm_rotary& a, void* dq, void* dk, float* dw_q, float* dw_k,
                                     void* workspace, hipStream_t stream) {
  const NormParams p = params(a);
  const int rows = static_cast<int>(blocks(p, kMaxBlocks));
  float* const partial = static_cast<float*>(workspace);
  by_variant(a, [&](auto type, auto gs, auto inter) {
    norm_rotary_bwd_kernel<decltype(type), gs.value, inter.value><<<rows, kThreads, 0, stream>>>(p, dq, dk, partial);
  });
  if (dw_q != nullptr || dw_k != nullptr)
    weight_sum_kernel<<<2 * p.D / 4, kThreads, 0, stream>>>(partial, rows, p.D, dw_q, dw_k);
  return hipGetLastError();
}

}  // namespace hz
