// Device helpers shared by the token attention kernels (include/hz_token.h).
//
// One kernel text serves both storage types: an operand of a product is PARTS registers quadruples of
// eight bfloat16, one for bfloat16 tensors, three for float32 ones (the split of split_f32.h, whose six
// products give float32's precision). Products are v_mfma_f32_32x32x16_bf16 with the layouts of
// split_f32.h: lane l = 32 hh + c.
//
// Scores are formed transposed, S^T = K Q^T (keys in a lane's sixteen registers, one query a lane), so
// a row's softmax is a sum over registers and one exchange with the other half wave, and a lane's
// weights of keys kappa(s, hh, j) = 16 s + 8 (j / 4) + 4 hh + j % 4, j = 0..7, are its B operand of the
// product with V's rows in that order, without moving a value between lanes.
//
// LDS tiles hold rows of DP bfloat16 in chunks of eight; chunk i of row r lies at chunk
// i ^ swizzle(r). Rows of one 256-byte line then differ where sixteen rows are read at one chunk (the
// A operand of K Q^T) and where four rows are read at four chunks (the transposing reads of the A
// operand V^T), so both go through without bank conflicts and without padding.
#pragma once

#include "mhsea_device.h"
#include "split_f32.h"
#include "token_launch.h"

namespace hz {
namespace token {

constexpr float kNegInf = -__builtin_inff();

struct Params {
  hz_token_tensor q, k, v;
  void *out, *out_low;
  float* lse;
  const float* slopes;
  const int32_t *prefix, *documents, *kv_len;
  const int *q_order, *k_order;  // the blocks of all rows, the longest first (null: in their own order)
  int B, Nq, Nk, H, Hk, G, D, causal;
  float scale;      // of the dot products
  float cap;        // 0: not capped
  float to_tanh;    // scale / cap
  float to_exp2;    // 2 log2 e scale / cap: e^2y = 2^(this x)
  float to_score2;  // base-2 score of a dot product (scale log2 e) or of a tanh (cap log2 e)
};

inline Params make_params(const hz_token_attention& a) {
  Params p{};
  p.q = a.q, p.k = a.k, p.v = a.v, p.out = a.out, p.out_low = a.out_low, p.lse = a.lse;
  p.slopes = a.slopes, p.prefix = a.prefix, p.documents = a.documents, p.kv_len = a.kv_len;
  p.B = static_cast<int>(a.B), p.Nq = static_cast<int>(a.Nq), p.Nk = static_cast<int>(a.Nk);
  p.H = static_cast<int>(a.H), p.Hk = static_cast<int>(a.Hk), p.G = p.H / p.Hk, p.D = static_cast<int>(a.D);
  p.causal = a.causal, p.scale = a.scale, p.cap = a.softcap;
  p.to_tanh = a.softcap > 0.f ? a.scale / a.softcap : 0.f;
  p.to_exp2 = 2.f * kLog2e * p.to_tanh;
  p.to_score2 = (a.softcap > 0.f ? a.softcap : a.scale) * kLog2e;
  return p;
}

// Eight consecutive elements in storage format, as loaded early and used late.
template <int PARTS>
struct Raw8;
template <>
struct Raw8<1> {
  v4u u;
  __device__ __forceinline__ void load(const void* base, int64_t off, bool on) {
    u = on ? *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(base) + off) : v4u{0u, 0u, 0u, 0u};
  }
};
template <>
struct Raw8<3> {
  v4f a, b;
  __device__ __forceinline__ void load(const void* base, int64_t off, bool on) {
    const v4f* const p = reinterpret_cast<const v4f*>(static_cast<const float*>(base) + off);
    a = on ? p[0] : zero4();
    b = on ? p[1] : zero4();
  }
};

__device__ __forceinline__ void floats(const Raw8<1>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(r.u[i] << 16);
    x[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void floats(const Raw8<3>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = r.a[i], x[4 + i] = r.b[i];
}

// An operand of eight bfloat16 a part.
template <int PARTS>
struct Frag {
  v4u p[PARTS];
};
__device__ __forceinline__ Frag<1> frag(const Raw8<1>& r) { return Frag<1>{{r.u}}; }
__device__ __forceinline__ Frag<3> frag(const Raw8<3>& r) {
  const float x[8] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3]};
  const Split8 s = split8(x);
  return Frag<3>{{s.h, s.m, s.l}};
}
// Elements 8 s .. 8 s + 7 of a score tile.
template <int PARTS>
__device__ __forceinline__ Frag<PARTS> frag_of(const v16f& x, int s) {
  if constexpr (PARTS == 1) {
    Frag<1> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.p[0][i] = pack2_bf16(x[8 * s + 2 * i], x[8 * s + 2 * i + 1]);
    return f;
  } else {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[8 * s + i];
    const Split8 f = split8(y);
    return Frag<3>{{f.h, f.m, f.l}};
  }
}

// The same for a score gradient. bfloat16: two parts, x cut to its upper half and the rest rounded, 2^-16 off together.
// In one part, dq and dk are off by 0.0025 of their size where their own rounding makes 0.0017 of it, and by up to 0.0028
// for short rows; in two by 0.0018. The second product costs 7% of the time (attn_train_packed_bf16 765 -> 817 us).
template <int PARTS>
__device__ __forceinline__ Frag<PARTS == 1 ? 2 : 3> grad_frag(const v16f& x, int s) {
  if constexpr (PARTS == 1) {
    Frag<2> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[8 * s + 2 * i], b = x[8 * s + 2 * i + 1];
      const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
      f.p[0][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302);
      f.p[1][i] = pack2_bf16(a - __builtin_bit_cast(float, ua & 0xffff0000u), b - __builtin_bit_cast(float, ub & 0xffff0000u));
    }
    return f;
  } else {
    return frag_of<3>(x, s);
  }
}

__device__ __forceinline__ v16f mma(const Frag<1>& a, const Frag<1>& b, v16f c) {
  return mfma32_bf16(as_bf16x8(a.p[0]), as_bf16x8(b.p[0]), c);
}
__device__ __forceinline__ v16f mma(const Frag<1>& a, const Frag<2>& b, v16f c) {
  c = mfma32_bf16(as_bf16x8(a.p[0]), as_bf16x8(b.p[1]), c);
  return mfma32_bf16(as_bf16x8(a.p[0]), as_bf16x8(b.p[0]), c);
}
__device__ __forceinline__ v16f mma(const Frag<3>& a, const Frag<3>& b, v16f c) {
#pragma unroll
  for (int t = 0; t < kSplitTerms; ++t) c = mfma32_bf16(as_bf16x8(a.p[kSplitA[t]]), as_bf16x8(b.p[kSplitB[t]]), c);
  return c;
}

// The product of the transposed operands (a takes b's place): the same terms in the same order, so that the sums of S and of S^T
// have the same bits.
__device__ __forceinline__ v16f mma_turned(const Frag<1>& a, const Frag<1>& b, v16f c) { return mma(a, b, c); }
__device__ __forceinline__ v16f mma_turned(const Frag<3>& a, const Frag<3>& b, v16f c) {
#pragma unroll
  for (int t = 0; t < kSplitTerms; ++t) c = mfma32_bf16(as_bf16x8(a.p[kSplitB[t]]), as_bf16x8(b.p[kSplitA[t]]), c);
  return c;
}

__device__ __forceinline__ v4f mma16(const Frag<1>& a, const Frag<1>& b, v4f c) {
  return mfma16_bf16(as_bf16x8(a.p[0]), as_bf16x8(b.p[0]), c);
}
__device__ __forceinline__ v4f mma16(const Frag<3>& a, const Frag<3>& b, v4f c) {
#pragma unroll
  for (int t = 0; t < kSplitTerms; ++t) c = mfma16_bf16(as_bf16x8(a.p[kSplitA[t]]), as_bf16x8(b.p[kSplitB[t]]), c);
  return c;
}

// Products are waited for here, before any branch: a vector instruction may read a product's result only some
// wait states after it, and where paths of different lengths lead from one to the other the compiler
// (ROCm 7.2's) counts them on one path only. Twenty wait states are more than the twelve that the 32 x 32 x 16
// product needs.
template <int N>
__device__ __forceinline__ void settle(v16f (&x)[N]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 3");
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[n]));
  __builtin_amdgcn_sched_barrier(0);
}
template <int M, int N>
__device__ __forceinline__ void settle(v4f (&x)[M][N]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 3");
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[m][n]));
  __builtin_amdgcn_sched_barrier(0);
}

// x, which the compiler takes for a new value: addresses formed from it are formed again where they are used
// and do not hold registers all through a loop.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// N steps of use(i, load(i)) with the next step's operands read from LDS ahead of each step's products: left alone, the
// compiler reads an operand right before the product that needs it and waits for LDS every time. (Three parts: six
// products an operand hide that wait, and the registers of a second one cost more: attn_train_sites_f32 3% slower.)
template <int N, int PARTS, class Load, class Use>
__device__ __forceinline__ void ahead(Load load, Use use) {
  if constexpr (PARTS == 3) {
#pragma unroll
    for (int i = 0; i < N; ++i) use(i, load(i));
    return;
  }
  auto now = load(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    auto next = now;
    if (i + 1 < N) next = load(i + 1);
    __builtin_amdgcn_sched_barrier(0);
    use(i, now);
    now = next;
  }
}

// A tile of ROWS rows of DP elements in LDS, PARTS planes.
template <int ROWS, int DP, int PARTS>
struct Tile {
  static constexpr int kPlane = ROWS * DP;
  static constexpr int kBytes = kPlane * PARTS * 2;
  uint16_t* base;

  __device__ __forceinline__ static int swizzle(int row) {
    const int low = (row >> 2) & 3;
    return DP == 128 ? ((row & 3) << 2) | low : DP == 64 ? (((row >> 1) & 1) << 2) | low : low;
  }
  __device__ __forceinline__ static int at(int row, int chunk) { return row * DP + ((chunk ^ swizzle(row)) << 3); }

  __device__ __forceinline__ void put(int row, int chunk, const Frag<PARTS>& f) const {
    const int o = at(row, chunk);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) *reinterpret_cast<v4u*>(base + i * kPlane + o) = f.p[i];
  }
  // A operand of a product over the columns: lane (hh, c) gets row row0 + c, elements 16 s + 8 hh .. + 7.
  __device__ __forceinline__ Frag<PARTS> rows(int row0, int s, int lane) const {
    const int o = at(row0 + (lane & 31), lane >> 5) ^ (s << 4);  // chunk 2 s + hh: s flips bits above hh's
    Frag<PARTS> f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) f.p[i] = *reinterpret_cast<const v4u*>(base + i * kPlane + o);
    return f;
  }
  // A operand of a product over the rows: lane (hh, c) gets column 32 dt + c of the rows row0 + 8 (j / 4)
  // + 4 hh + j % 4, j = 0..7. Lane 16 g + 4 j + q addresses row 4 (g / 2) + j (then eight rows on),
  // columns 32 dt + 16 (g % 2) + 4 q .. + 3; the hardware transposes the 16-lane groups. row0 is a
  // multiple of 16.
  __device__ __forceinline__ Frag<PARTS> columns(int row0, int dt, int lane) const {
    typedef short v4s __attribute__((ext_vector_type(4)));
    const int g = lane >> 4, m = lane & 15, row = row0 + 4 * (g >> 1) + (m >> 2);
    const int o0 = (at(row, 2 * (g & 1) + ((m & 3) >> 1)) ^ (dt << 5)) + 4 * (m & 1);  // chunk 4 dt + ..
    const int o1 = (o0 ^ 16) + 8 * DP;  // eight rows on, the swizzle differs in one bit
    Frag<PARTS> f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(base + i * kPlane + o0));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(base + i * kPlane + o1));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      f.p[i] = v4u{l.x, l.y, h.x, h.y};
    }
    return f;
  }
  // The same for the 16 x 16 x 32 product over 32 rows: lane 16 g + c gets column 16 dt + c of the rows
  // 16 (j / 4) + 4 g + j % 4.
  __device__ __forceinline__ Frag<PARTS> columns16(int dt, int lane) const {
    typedef short v4s __attribute__((ext_vector_type(4)));
    const int g = lane >> 4, m = lane & 15, row = 4 * g + (m >> 2);
    const int o0 = (at(row, (m & 3) >> 1) ^ (dt << 4)) + 4 * (m & 1);  // chunk 2 dt + ..
    const int o1 = o0 + 16 * DP;  // the swizzle repeats after sixteen rows
    Frag<PARTS> f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(base + i * kPlane + o0));
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(base + i * kPlane + o1));
      const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
      f.p[i] = v4u{l.x, l.y, h.x, h.y};
    }
    return f;
  }
};

// tanh by 1 - 2 / (1 + e^2y). Its error, an absolute 1e-7, is a relative one of small scores and grows by the cap, so
// float32 tensors get y + y z P(z), z = y^2, below 3/4: P is fitted to (tanh(y) / y - 1) / z at the Chebyshev points of
// 0 <= z <= 9/16, 7e-9 of the result off, 7e-8 with its roundings.
template <int PARTS>
__device__ __forceinline__ float tanh_of(float y) {
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + fast_exp2(2.f * kLog2e * y));
  if constexpr (PARTS == 1) return big;
  const float z = y * y;
  float s = 0.00191453761f;
  s = fmaf(s, z, -0.00794092473f);
  s = fmaf(s, z, 0.0216188449f);
  s = fmaf(s, z, -0.0539365672f);
  s = fmaf(s, z, 0.13333185f);
  s = fmaf(s, z, -0.333333313f);
  return fabsf(y) < 0.75f ? fmaf(y, z * s, y) : big;
}

// Element i of a lane's sixteen scores of a 32-row block belongs to row 8 (i / 4) + 4 hh + i % 4.
__device__ __forceinline__ int row_of(int i, int hh) { return 8 * (i >> 2) + 4 * hh + (i & 3); }

__device__ __forceinline__ int kv_length(const Params& p, int b) {
  if (p.kv_len == nullptr) return p.Nk;
  const int n = p.kv_len[b];
  return n < 0 ? 0 : n > p.Nk ? p.Nk : n;
}

// What one query may see: keys up to `last`, and where there are documents those of `doc`.
constexpr int kNoDocument = -2147483647 - 1;
struct Sight {
  int pos, last, doc;
  Sight() = default;
  __device__ __forceinline__ Sight(const Params& p, int b, int i, int n) {
    pos = n - p.Nq + i;
    last = n - 1;
    if (p.causal) {
      const int pre = p.prefix != nullptr ? max(p.prefix[b], 0) : 0;
      const int near = max(pos, pre - 1);
      last = near < last ? near : last;
    }
    doc = kNoDocument;
    if (p.documents != nullptr && pos >= 0) {
      const int d = p.documents[static_cast<int64_t>(b) * p.Nk + pos];
      doc = d >= 0 ? d : kNoDocument;
    }
  }
};
// A key's document, with every padding number the same.
__device__ __forceinline__ int key_document(const Params& p, int b, int j) {
  const int d = p.documents[static_cast<int64_t>(b) * p.Nk + j];
  return d >= 0 ? d : -1;
}

// Documents of 64 consecutive keys: the smallest and largest number among them (lo > hi: none), and
// whether any of the 64 is padding or behind the row's end.
struct DocTile {
  int lo, hi, pad, unused;
};
constexpr int kDocTile = 64;

// Which unit of work a workgroup takes: `inner` workgroups on each key head of a block of 128 rows, for one block after
// the other, so that every XCD (workgroups go round the 8 by their number) gets its share of the long blocks. Blocks
// are taken in `order` where there is one, else the last or first of every row before the next. (Pairs of row and
// key head kept on XCDs of their own, for their L2, were no faster forward and 3 to 10% slower in reverse:
// attn_train_packed_bf16 761 us so, 787 to 836 with pairs on XCDs.)
struct Unit {
  int inner, hk, b, tile;
  __device__ __forceinline__ Unit(const Params& p, int64_t id, int inner_, int tiles, bool last_first, const int* order) {
    inner = static_cast<int>(id % inner_);
    id /= inner_;
    hk = static_cast<int>(id % p.Hk);
    id /= p.Hk;
    if (order != nullptr) {
      const int e = order[id];
      b = e / tiles;
      tile = e - b * tiles;
    } else {
      b = static_cast<int>(id % p.B);
      const int t = static_cast<int>(id / p.B);
      tile = last_first ? tiles - 1 - t : t;
    }
  }
};

// Copies rows of a strided tensor straight into a Tile of bfloat16 (16 bytes a lane, no registers): what a lane
// reads is chosen so that lane i's 16 bytes land where the tile wants them. Rows behind the last one
// repeat it and chunks behind D repeat the first: finite, and multiplied by zeros.
template <int ROWS, int DP>
struct Copy {
  static constexpr int CH = DP / 8, LOADS = ROWS * CH / 256;
  const uint16_t *base, *mine;  // the head's first row at this lane's chunk; this lane's row of the first tile
  int64_t token;
  int row, wave;  // this lane's row in the first of LOADS parts; STEP rows between parts
  static constexpr int STEP = 256 / CH;
  __device__ __forceinline__ Copy(const hz_token_tensor& t, int64_t b, int64_t h, int D, int tid) {
    row = tid / CH;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunk = (tid % CH) ^ Tile<ROWS, DP, 1>::swizzle(row);
    base = static_cast<const uint16_t*>(t.data) + b * t.batch + h * t.head + (8 * chunk < D ? 8 * chunk : 0);
    token = t.token;
    mine = base + row * token;
  }
  __device__ __forceinline__ void operator()(uint16_t* lds, int r0, int rows) const {
    if (r0 + ROWS <= rows) {  // one addition of a scalar an address
#pragma unroll
      for (int j = 0; j < LOADS; ++j) one(lds, j, mine + (r0 + STEP * j) * token);
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) one(lds, j, base + static_cast<int64_t>(min(r0 + row + STEP * j, rows - 1)) * token);
    }
  }
  __device__ __forceinline__ void one(uint16_t* lds, int j, const uint16_t* src) const {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)(lds + (4 * j + wave) * 512), 16, 0, 0);
  }
};
// The copies issued so far have landed in LDS for every wave that passes the barrier behind this.
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The tiles of KB rows that a block has to visit, in order: all of [begin, end), or with documents those
// whose range of numbers meets the block's. One load and one vote decide 64 tiles.
template <class Range>
struct Walk {
  int begin, end, group;
  uint64_t votes;
  DocTile mine;
  bool by_document;
  Range range;  // tile index -> DocTile
  int lo, hi;
  __device__ __forceinline__ Walk(int begin_, int end_, bool by_document_, int lo_, int hi_, Range range_)
      : begin(begin_), end(end_), group(-1), votes(0), mine{}, by_document(by_document_), range(range_), lo(lo_), hi(hi_) {}
  // Narrows [begin, end) to the first and last tile to visit, and then to one of n equal parts.
  __device__ __forceinline__ void take_part(int part, int n, int lane) {
    if (by_document) {
      DocTile doc;
      begin = next(begin, lane, doc);
      int last = begin;
      for (int g = end > 0 ? (end - 1) & ~63 : -1; g >= begin - 63 && begin < end; g -= 64) {
        const DocTile x = g + lane < end ? range(g + lane) : DocTile{2147483647, -1, 1, 0};
        const uint64_t v = __ballot(x.lo <= hi && x.hi >= lo);
        if (v != 0) {
          last = g + 64 - __clzll(static_cast<long long>(v));
          break;
        }
      }
      end = max(begin, last);
      group = -1;
    }
    const int64_t count = end - begin;
    const int first = begin;
    begin = first + static_cast<int>(count * part / n);
    end = first + static_cast<int>(count * (part + 1) / n);
  }
  // The first tile >= t to visit (end: none), and its documents.
  __device__ __forceinline__ int next(int t, int lane, DocTile& doc) {
    if (!by_document) return t;
    while (t < end) {
      const int g = t & ~63;
      if (g != group) {
        group = g;
        mine = DocTile{2147483647, -1, 1, 0};
        if (g + lane < end) mine = range(g + lane);
        votes = __ballot(mine.lo <= hi && mine.hi >= lo);
      }
      const uint64_t rest = votes >> (t - g);
      if (rest != 0) {
        t += __ffsll(static_cast<unsigned long long>(rest)) - 1;
        if (t >= end) return end;
        doc.lo = __builtin_amdgcn_readlane(mine.lo, t - g);
        doc.hi = __builtin_amdgcn_readlane(mine.hi, t - g);
        doc.pad = __builtin_amdgcn_readlane(mine.pad, t - g);
        return t;
      }
      t = g + 64;
    }
    return end;
  }
};

// Smallest and largest document of a wave's queries; lo > hi if it has none.
__device__ __forceinline__ void document_range(int doc, int& lo, int& hi) {
  lo = doc >= 0 ? doc : 2147483647;
  hi = doc >= 0 ? doc : -1;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    lo = min(lo, __shfl_xor(lo, x, 64));
    hi = max(hi, __shfl_xor(hi, x, 64));
  }
}

// Four consecutive elements in the tensor's type.
template <int PARTS>
__device__ __forceinline__ void store_four(void* out, int64_t off, float a, float b, float c, float d) {
  if constexpr (PARTS == 1)
    store4<BF16>(out, off, a, b, c, d);
  else
    store4<F32>(out, off, a, b, c, d);
}

// Into how many parts the n rows that a kernel streams are divided so that its `blocks` workgroups become about `want`;
// a part has at least 128 rows.
inline int share_of(int64_t blocks, int64_t n, int64_t want) {
  const int64_t wanted = want / blocks, most = n / 128, parts = wanted < most ? wanted : most;
  return static_cast<int>(parts > 1 ? parts : 1);
}

// The passes over the documents (token_attention_fwd.hip), where a call has some: the DocTiles at `memory`, and the
// order of the blocks of queries, and of keys, behind them.
constexpr int kOrderBlock = 128;  // rows of a block
int64_t doc_bytes(const hz_token_attention& a);
hipError_t launch_docs(const hz_token_attention& a, Params& p, bool keys, void* memory, hipStream_t stream);

}  // namespace token
}  // namespace hz
