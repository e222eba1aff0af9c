// Norms of queries and keys for each head with the position rotation in the same pass, and their
// reverse mode (formulas: include/hz_token.h).
//
// One head of D elements is held by L = D / 8 lanes, eight elements a lane as two chunks of four,
// chosen so that both elements of each rotated pair are in one lane and no lane exchanges data but
// for the sum of squares: with half-split pairs lane t holds elements 4 t .. 4 t + 3 and
// n_freqs + 4 t .. + 3, with interleaved ones (and behind the rotated part) 8 t .. 8 t + 7. Either
// way it turns pairs 4 t .. 4 t + 3. A workgroup takes a few tokens at a time: it forms their angles
// once, in float64 turns (an angle at position 10^5 has no bits to lose in float32's 24), puts the sines
// and cosines into LDS, and then runs over the tokens' query and key heads, the next ones' data in flight
// while one is normalised. With several axes each pair has its axis' position; the rest is the same.
// x is read and y written once; the backward reads x and dy and writes dx. float32: bound by those bytes (256 x 225 tokens of 16
// heads of 64: 112 us, 5.0 TB/s, and 140 in reverse mode, 5.2 TB/s); bfloat16: by vector instructions beside them (4 x
// 4096 tokens of 40 heads of 128: 84 us, 4.0 TB/s, and 117 us, 4.3 TB/s).
#include "mhsea_device.h"
#include "paged_launch.h"
#include "token_launch.h"

namespace hz {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;    // a workgroup at a time, forward
constexpr int kMaxTokensBwd = 4;   // and backward
constexpr int kMaxBlocks = 1024;  // of the backward: rows of partial weight gradients

struct NormParams {
  hz_token_tensor q, k, qo, ko;
  const float *wq, *wk;
  const double* freqs;
  const int32_t *positions, *axes;  // positions of n_axes a token; axes null: the first
  int64_t tokens;
  int N, H, HT, D, nf, n_axes, interleaved, each;  // each: tokens a workgroup at a time
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

typedef float2 Angles[HZ_ROTARY_MAX_HEAD / 2];  // of a token

__device__ __forceinline__ void put_angles(const NormParams& p, int64_t token0, int count, Angles* angles) {
  for (int a = threadIdx.x; a < count * p.nf; a += kThreads) {
    const int x = a / p.nf, f = a - x * p.nf;
    const int64_t token = token0 + x;
    const int axis = p.axes != nullptr ? p.axes[f] : 0;
    const bool known = axis >= 0 && axis < p.n_axes;  // a pair of no axis stays as it is
    const double pos = !known ? 0 : p.positions != nullptr ? p.positions[token * p.n_axes + axis] : static_cast<int>(token % p.N);
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

// The first of the tokens at hand: one 64-bit division for all of them.
struct First {
  int64_t b;
  int n;
  __device__ __forceinline__ First(const NormParams& p, int64_t token0) : b(token0 / p.N), n(static_cast<int>(token0 - b * p.N)) {}
};

// One (token, head) of the tokens at hand: which tensor, and where its head lies in the strided ones and in
// a contiguous one.
struct Item {
  bool is_q;
  int token, head, n;
  int64_t b;
  __device__ __forceinline__ Item(const NormParams& p, const First& first, int i) : Item(p, first, i / p.HT, i % p.HT) {}
  __device__ __forceinline__ Item(const NormParams& p, const First& first, int token_, int h)
      : is_q(h < p.H), token(token_), head(h < p.H ? h : h - p.H), n(first.n + token_), b(first.b) {
    while (n >= p.N) n -= p.N, ++b;  // (a few tokens)
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
  __shared__ Angles angles[kMaxTokens];
  constexpr int SLOTS = kThreads / GS;
  const int t = threadIdx.x % GS, slot = threadIdx.x / GS;
  const Lane lane(p, t);
  float wq[8], wk[8];
  weights(p.wq, lane, wq);
  weights(p.wk, lane, wk);
  for (int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.each; token0 < p.tokens;
       token0 += static_cast<int64_t>(gridDim.x) * p.each) {
    const int count = static_cast<int>(p.tokens - token0 < p.each ? p.tokens - token0 : p.each), items = count * p.HT;
    const First first(p, token0);
    Raw<S> next[2];
    auto load = [&](int i, int k) __attribute__((always_inline)) {
      if (i < items && lane.on) {
        const Item it(p, first, i);
        next[k].load(it.data(p.q, p.k), it.offset(p.q, p.k), lane);
      }
    };
    load(slot, 0);
    load(slot + SLOTS, 1);
    put_angles(p, token0, count, angles);
    __syncthreads();
    auto use = [&](int i, int k) __attribute__((always_inline)) {
      const Item it(p, first, i);
      float x[8];
      next[k].get(x, lane.on);
      load(i + 2 * SLOTS, k);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
      const float r = 1.f / sqrtf(head_sum<GS>(ss) / static_cast<float>(p.D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * (it.is_q ? wq[e] : wk[e]);
      if (lane.turns) turn8<INTERLEAVED>(x, &angles[it.token][4 * t], 1.f);
      if (lane.on) store8<S>(const_cast<void*>(it.data(p.qo, p.ko)), it.offset(p.qo, p.ko), lane, x);
    };
    for (int i = slot; i < items; i += 2 * SLOTS) {
      use(i, 0);
      if (i + SLOTS < items) use(i + SLOTS, 1);
    }
    __syncthreads();
  }
}

// q and k: the forward's inputs; qo and ko: the cotangents. partial: [gridDim.x][2][D]. Four workgroups a CU, so that all of the grid are
// there at once (float32 had registers for three: 157 us for 256 x 225 tokens of 16 heads of 64; with four, heads of more than 16
// elements spill two to four registers and take 140).
template <class S, int GS, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) norm_rotary_bwd_kernel(NormParams p, void* dq, void* dk, float* partial) {
  __shared__ Angles angles[kMaxTokensBwd];
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
    const First first(p, token0);
    Raw<S> next_x, next_g;
    auto load = [&](int i) {
      if (i < items && lane.on) {
        const Item it(p, first, i);
        next_x.load(it.data(p.q, p.k), it.offset(p.q, p.k), lane);
        next_g.load(it.data(p.qo, p.ko), it.offset(p.qo, p.ko), lane);
      }
    };
    load(slot);
    put_angles(p, token0, count, angles);
    __syncthreads();
    for (int i = slot; i < items; i += SLOTS) {
      const Item it(p, first, i);
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

// U elements of a head as they lie in memory.
template <class S, int U>
struct Chunk;
template <>
struct Chunk<F32, 4> {
  typedef uint32_t V __attribute__((ext_vector_type(4)));
  V v;
  __device__ __forceinline__ void get(float (&x)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
  }
  __device__ __forceinline__ void set(const float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(x[i]);
  }
};
template <int U>
struct Chunk<BF16, U> {
  typedef uint32_t V __attribute__((ext_vector_type(U / 2)));
  V v;
  __device__ __forceinline__ void get(float (&x)[U]) const {
#pragma unroll
    for (int i = 0; i < U / 2; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
  __device__ __forceinline__ void set(const float (&x)[U]) {
#pragma unroll
    for (int i = 0; i < U / 2; ++i) v[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
  }
};

// The rotation alone, from q and k to qo and ko, and back (dir -1), which is its reverse mode. A thread has two chunks of U elements of one
// head after the other, two heads in flight: a chunk and the one that it turns with (behind the rotated part: the next), or
// with interleaved pairs one in each half of the head, so that a wave's 16 bytes lie one behind the other. They are read once,
// past the caches (2 x 8160 tokens of 40 bfloat16 heads of 128: 60 us, 66 through them; 76 with chunks of 4, as behind the norms).
// Bound by those bytes: 5.6 TB/s.
template <class S, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(NormParams p, float dir) {
  __shared__ Angles angles[kMaxTokens];
  typedef typename S::T T;
  typedef typename Chunk<S, U>::V V;
  const int units = p.D / (2 * U), slots = kThreads / units, t = static_cast<int>(threadIdx.x) % units, slot = static_cast<int>(threadIdx.x) / units;
  const bool turns = U * t < p.nf;
  const int o0 = INTERLEAVED || turns ? U * t : 2 * U * t, o1 = INTERLEAVED ? p.D / 2 + U * t : turns ? p.nf + U * t : o0 + U;
  const int step_token = slots / p.HT, step_head = slots % p.HT;  // from a slot's item to its next
  for (int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.each; token0 < p.tokens;
       token0 += static_cast<int64_t>(gridDim.x) * p.each) {
    const int count = static_cast<int>(p.tokens - token0 < p.each ? p.tokens - token0 : p.each);
    const First first(p, token0);
    struct At {
      int token, head;
    };
    auto after = [&](At a) {
      a.token += step_token, a.head += step_head;
      if (a.head >= p.HT) a.head -= p.HT, ++a.token;
      return a;
    };
    Chunk<S, U> x[2], y[2];
    auto load = [&](At a, int i) __attribute__((always_inline)) {
      if (a.token >= count) return;
      const Item it(p, first, a.token, a.head);
      const T* const from = static_cast<const T*>(it.data(p.q, p.k)) + it.offset(p.q, p.k);
      x[i].v = __builtin_nontemporal_load(reinterpret_cast<const V*>(from + o0));
      y[i].v = __builtin_nontemporal_load(reinterpret_cast<const V*>(from + o1));
    };
    auto use = [&](At a, int i) __attribute__((always_inline)) {
      const Item it(p, first, a.token, a.head);
      float u[U], v[U];
      x[i].get(u), y[i].get(v);
      auto turn = [&](float& p0, float& p1, float2 angle) __attribute__((always_inline)) {
        const float c = angle.x, s = dir * angle.y, m = p0, n = p1;
        p0 = m * c - n * s;
        p1 = n * c + m * s;
      };
      if constexpr (INTERLEAVED) {
        auto pairs = [&](Chunk<S, U>& chunk, float (&w)[U], int pair) __attribute__((always_inline)) {
          if (pair >= p.nf) return;
#pragma unroll
          for (int e = 0; e < U / 2; ++e) turn(w[2 * e], w[2 * e + 1], angles[a.token][pair + e]);
          chunk.set(w);
        };
        pairs(x[i], u, o0 / 2);
        pairs(y[i], v, o1 / 2);
      } else if (turns) {
#pragma unroll
        for (int e = 0; e < U; ++e) turn(u[e], v[e], angles[a.token][U * t + e]);
        x[i].set(u), y[i].set(v);
      }
      T* const to = static_cast<T*>(const_cast<void*>(it.data(p.qo, p.ko))) + it.offset(p.qo, p.ko);
      *reinterpret_cast<V*>(to + o0) = x[i].v;
      *reinterpret_cast<V*>(to + o1) = y[i].v;
    };
    At a{slot / p.HT, slot % p.HT}, b = after(a);
    if (slot >= slots) a.token = b.token = count;
    load(a, 0);
    load(b, 1);
    put_angles(p, token0, count, angles);
    __syncthreads();
    while (a.token < count) {
      use(a, 0);
      a = after(b);
      load(a, 0);
      if (b.token >= count) break;
      use(b, 1);
      b = after(a);
      load(b, 1);
    }
    __syncthreads();
  }
}

// Tokens a workgroup at a time: several where that leaves at least `blocks` workgroups, so that the angles are
// formed by all lanes and the loads of several heads overlap (the forwards of
// qk_train_bf16 and qk_train_sites_f32: 90 and 93 us, 115 and 220 with one token), at most `most`. Forward that is the largest power of two up to 16
// whose tokens have 160 heads or fewer in all, or one token (2 x 8160 tokens of 40 heads, 4 and 16 tokens a time: 61 us, 73; 256 x 225 of 16
// heads, 4 and 8: 52 and 50, behind norms 116 and 112).
int tokens_each(int64_t tokens, int64_t blocks, int most) {
  const int64_t n = tokens / blocks;
  return static_cast<int>(n < 1 ? 1 : n > most ? most : n);
}
int forward_each(const NormParams& p) {
  int n = kMaxTokens;
  while (n > 1 && n * p.HT > 160) n /= 2;
  return tokens_each(p.tokens, kMaxBlocks, n);
}

NormParams params(const hz_qk_norm_rotary& a) {
  NormParams p{};
  p.q = a.q, p.k = a.k, p.qo = a.q_out, p.ko = a.k_out;
  p.wq = a.w_q, p.wk = a.w_k, p.freqs = a.freqs, p.positions = a.positions;
  p.tokens = a.B * a.N;
  p.N = static_cast<int>(a.N), p.H = static_cast<int>(a.H), p.HT = static_cast<int>(a.H + a.Hk);
  p.D = static_cast<int>(a.D), p.nf = static_cast<int>(a.n_freqs), p.interleaved = a.interleaved, p.n_axes = 1;
  p.each = tokens_each(p.tokens, kMaxBlocks, kMaxTokensBwd);
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

NormParams params(const hz_qk_rotary& a) {
  NormParams p = params(a.rotary);
  p.axes = a.axes, p.n_axes = static_cast<int>(a.n_axes);
  if (!a.norm) p.wq = p.wk = nullptr;
  return p;
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

hipError_t run_fwd(NormParams p, const hz_qk_norm_rotary& a, hipStream_t stream) {
  p.each = forward_each(p);
  const dim3 grid(static_cast<unsigned>(blocks(p, 1 << 20)));
  by_variant(a, [&](auto type, auto gs, auto inter) {
    norm_rotary_fwd_kernel<decltype(type), gs.value, inter.value><<<grid, kThreads, 0, stream>>>(p);
  });
  return hipGetLastError();
}

hipError_t run_rotary(NormParams p, float dir, int32_t dtype, hipStream_t stream) {
  p.each = forward_each(p);
  const dim3 grid(static_cast<unsigned>(blocks(p, 1 << 20)));
  auto run = [&](auto type, auto u) {
    if (p.interleaved)
      rotary_kernel<decltype(type), u.value, true><<<grid, kThreads, 0, stream>>>(p, dir);
    else
      rotary_kernel<decltype(type), u.value, false><<<grid, kThreads, 0, stream>>>(p, dir);
  };
  if (dtype == HZ_DTYPE_F32)
    run(F32{}, std::integral_constant<int, 4>{});
  else if (p.D % 16 == 0 && p.nf % 8 == 0)
    run(BF16{}, std::integral_constant<int, 8>{});
  else
    run(BF16{}, std::integral_constant<int, 4>{});
  return hipGetLastError();
}

hipError_t run_bwd(const NormParams& p, const hz_qk_norm_rotary& a, void* dq, void* dk, float* dw_q, float* dw_k,
                   void* workspace, hipStream_t stream) {
  const int rows = static_cast<int>(blocks(p, kMaxBlocks));
  float* const partial = static_cast<float*>(workspace);
  by_variant(a, [&](auto type, auto gs, auto inter) {
    norm_rotary_bwd_kernel<decltype(type), gs.value, inter.value><<<rows, kThreads, 0, stream>>>(p, dq, dk, partial);
  });
  if (dw_q != nullptr || dw_k != nullptr)
    weight_sum_kernel<<<2 * p.D / 4, kThreads, 0, stream>>>(partial, rows, p.D, dw_q, dw_k);
  return hipGetLastError();
}

}  // namespace

int64_t qk_norm_rotary_workspace(int64_t tokens, int64_t D) {
  return (tokens < kMaxBlocks ? tokens : kMaxBlocks) * 2 * D * static_cast<int64_t>(sizeof(float));
}

hipError_t launch_qk_norm_rotary_fwd(const hz_qk_norm_rotary& a, hipStream_t stream) {
  return run_fwd(params(a), a, stream);
}

hipError_t launch_qk_norm_rotary_bwd(const hz_qk_norm_rotary& a, void* dq, void* dk, float* dw_q, float* dw_k,
                                     void* workspace, hipStream_t stream) {
  return run_bwd(params(a), a, dq, dk, dw_q, dw_k, workspace, stream);
}

int64_t qk_rotary_workspace(int64_t tokens, int64_t D, bool norm) { return norm ? qk_norm_rotary_workspace(tokens, D) : 0; }

hipError_t launch_qk_rotary_fwd(const hz_qk_rotary& a, hipStream_t stream) {
  const NormParams p = params(a);
  return a.norm ? run_fwd(p, a.rotary, stream) : run_rotary(p, 1.f, a.rotary.dtype, stream);
}

hipError_t launch_qk_rotary_bwd(const hz_qk_rotary& a, void* dq, void* dk, float* dw_q, float* dw_k, void* workspace,
                                hipStream_t stream) {
  NormParams p = params(a);
  if (a.norm) return run_bwd(p, a.rotary, dq, dk, dw_q, dw_k, workspace, stream);
  p.q = p.qo, p.k = p.ko;
  p.qo = {dq, static_cast<int64_t>(p.N) * p.H * p.D, static_cast<int64_t>(p.H) * p.D, p.D};
  p.ko = {dk, static_cast<int64_t>(p.N) * (p.HT - p.H) * p.D, static_cast<int64_t>(p.HT - p.H) * p.D, p.D};
  return run_rotary(p, -1.f, a.rotary.dtype, stream);
}

}  // namespace hz
