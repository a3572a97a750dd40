// Kernels of a layer's attention side over an 8-bit cache, for gfx950:
// per-head RMSNorm with the position rotation, the store into the cache,
// reading it back, and causal attention over it.
#include "kv8.h"

#include <stdint.h>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int BLK = FMA_KV8_BLOCK;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSplits = 128;
constexpr float kMinAmax = 7.888609052210118e-31f;  // 2^-100

// ---------------------------------------------------------------------------
// types

struct Bf16 {
  typedef uint16_t raw;
  static constexpr uint32_t kInf = 0x7f80, kMaxFinite = 0x7f7f;
  static constexpr float kMost = 3.3895313892515355e38f;
  static constexpr float kFine = 1.0f;
  static __device__ float to_f(uint16_t u) {
    return __uint_as_float(static_cast<uint32_t>(u) << 16);
  }
  static __device__ uint16_t from_f(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
  }
};
struct Fp16 {
  typedef uint16_t raw;
  static constexpr uint32_t kInf = 0x7c00, kMaxFinite = 0x7bff;
  static constexpr float kMost = 65504.0f;
  static constexpr float kFine = 16384.0f;  // keeps a second part's bits
  static __device__ float to_f(uint16_t u) {
    return static_cast<float>(__builtin_bit_cast(_Float16, u));
  }
  static __device__ uint16_t from_f(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
};
struct Fp32 {
  typedef float raw;
  static __device__ float to_f(float f) { return f; }
  static __device__ float from_f(float f) { return f; }
};

// Eight values of a row from d0 on; what lies behind hd comes as zero.
__device__ inline u16x8 load_raw(const uint16_t* row, int d0, int hd,
                                 bool vec) {
  u16x8 u = {0, 0, 0, 0, 0, 0, 0, 0};
  if (d0 >= hd) return u;
  if (vec) return *reinterpret_cast<const u16x8*>(row + d0);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (d0 + j < hd) u[j] = row[d0 + j];
  return u;
}
template <typename E>
__device__ inline void load8(const typename E::raw* row, int d0, int hd,
                             bool vec, float (&x)[8]) {
  if (d0 >= hd) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.0f;
    return;
  }
  if constexpr (sizeof(typename E::raw) == 2) {
    if (vec) {
      const u16x8 u = *reinterpret_cast<const u16x8*>(row + d0);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = E::to_f(u[j]);
      return;
    }
  } else {
    if (vec) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(row + d0);
      const f32x4 b = *reinterpret_cast<const f32x4*>(row + d0 + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = a[j];
        x[4 + j] = b[j];
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = d0 + j < hd ? E::to_f(row[d0 + j]) : 0.0f;
}

// PAST: past the caches, for outputs larger than they are.
template <bool PAST, typename V>
__device__ inline void put(void* at, V v) {
  if constexpr (PAST)
    __builtin_nontemporal_store(v, static_cast<V*>(at));
  else
    *static_cast<V*>(at) = v;
}
template <typename E, bool PAST>
__device__ inline void store8(typename E::raw* row, int d0, int hd, bool vec,
                              const float (&x)[8]) {
  if (d0 >= hd) return;
  if constexpr (sizeof(typename E::raw) == 2) {
    if (vec) {
      u16x8 u;
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = E::from_f(x[j]);
      put<PAST>(row + d0, u);
      return;
    }
  } else {
    if (vec) {
      put<PAST>(row + d0, f32x4{x[0], x[1], x[2], x[3]});
      put<PAST>(row + d0 + 4, f32x4{x[4], x[5], x[6], x[7]});
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (d0 + j < hd) row[d0 + j] = E::from_f(x[j]);
}

// ---------------------------------------------------------------------------
// Norm and rotation of one head.
//   y = x * rsqrt(mean(x^2) + eps) * w;  (a, b) -> (a c - b s, a s + b c)
// A row is held by LPR neighbouring lanes, eight values each, so the mean is
// log2(LPR) shuffles and pairs (2i, 2i+1) turn inside a lane; the two-halves
// layout takes its partners from another lane, or through LDS where they are
// not all one lane's. All in fp32 with one rounding at the end. The tables
// are read once for all heads that a row of lanes takes.
//
// Bound by memory: 8192 tokens of 32 + 8 heads of 128 in bf16 (172 MB) take
// 33.6 us, 5.1 TB/s, what a copy of 1 GiB reaches. One token is a launch.

template <int LPR>
__device__ inline float lanes_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

template <int LPR, bool PAIRS>
struct Turn {
  float c[8], s[8];  // of each of the lane's values; s signed in halves
  float w[8];
  bool norm;
  bool bad;  // position outside the table

  // the tables' rows at `pos`; lane holds values d0..d0+7
  __device__ void at(const FmaRope& r, long long pos, int d0) {
    bad = r.table > 0 && (pos < 0 || pos >= r.table);
    const bool on = r.table > 0 && !bad;
    const float* ct = r.cos + (on ? pos * r.half : 0);
    const float* st = r.sin + (on ? pos * r.half : 0);
    if (PAIRS && r.tab_vec) {
      // all four of a lane's pairs turn, or none
      f32x4 cv = {1, 1, 1, 1}, sv = {0, 0, 0, 0};
      if (on && d0 / 2 < r.half) {
        cv = *reinterpret_cast<const f32x4*>(ct + d0 / 2);
        sv = *reinterpret_cast<const f32x4*>(st + d0 / 2);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j] = cv[j];
        s[j] = sv[j];
      }
    } else if (!PAIRS && r.tab_vec && r.half % 8 == 0) {
      // a lane's values are all in one half, or behind both
      const bool in = on && d0 < 2 * r.half;
      const int i = d0 < r.half ? d0 : d0 - r.half;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        f32x4 cv = {1, 1, 1, 1}, sv = {0, 0, 0, 0};
        if (in) {
          cv = *reinterpret_cast<const f32x4*>(ct + i + 4 * n);
          sv = *reinterpret_cast<const f32x4*>(st + i + 4 * n);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[4 * n + j] = cv[j];
          s[4 * n + j] = d0 < r.half ? -sv[j] : sv[j];
        }
      }
    } else if constexpr (PAIRS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = d0 / 2 + j;
        const bool in = on && i < r.half;
        c[j] = in ? ct[i] : 1.0f;
        s[j] = in ? st[i] : 0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        const bool in = on && d < 2 * r.half;
        const int i = d < r.half ? d : d - r.half;
        c[j] = in ? ct[i] : 1.0f;
        const float sv = in ? st[i] : 0.0f;
        s[j] = d < r.half ? -sv : sv;
      }
    }
  }

  template <typename E>
  __device__ void weights(const void* p, int d0, int hd, bool vec) {
    norm = p != nullptr;
    if (norm)
      load8<E>(static_cast<const typename E::raw*>(p), d0, hd, vec, w);
  }

  // scratch: LPR * 8 floats of this row of lanes. The fused multiply-adds
  // are written out, so that every kernel that runs this gives the same bits.
  __device__ void run(float (&x)[8], const FmaRope& r, int hd, int d0,
                      float* scratch) const {
#pragma clang fp contract(off)
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
      const float rs =
          rsqrtf(lanes_sum<LPR>(ss) / static_cast<float>(hd) + r.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * rs * w[j];
    }
    if (r.table == 0) return;
    if constexpr (PAIRS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (d0 / 2 + j < r.half) {
          const float a = x[2 * j], b = x[2 * j + 1];
          x[2 * j] = fmaf(a, c[j], -(b * s[j]));
          x[2 * j + 1] = fmaf(a, s[j], b * c[j]);
        }
      }
    } else if ((r.half & 7) == 0) {
      // the partners of a lane's values are one other lane's
      const int by = r.half >> 3, li = d0 >> 3;
      const int from = (threadIdx.x & 63) + (li < by ? by : -by);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = __shfl(x[j], from);
        if (d0 < 2 * r.half) x[j] = fmaf(x[j], c[j], y * s[j]);
      }
    } else {
      // value d of the row lies at [d % 8][d / 8]: neighbouring lanes on
      // neighbouring banks
      const int li = d0 / 8;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 8; ++j) scratch[j * LPR + li] = x[j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        if (d < 2 * r.half) {
          const int p = d < r.half ? d + r.half : d - r.half;
          x[j] = fmaf(x[j], c[j], scratch[(p & 7) * LPR + (p >> 3)] * s[j]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (bad) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(0x7fc00000u);
    }
  }
};

__device__ inline long long pos_of(const FmaPos& p, int b, int t) {
  if (p.p32 == nullptr && p.p64 == nullptr) return p.start + t;
  const long long i = b * p.sb + (p.per_token ? t * p.st : 0);
  const long long v = p.p32 != nullptr ? p.p32[i] : p.p64[i];
  return p.per_token ? v : v + t;
}

// Heads [h0, h1) of one token, one after the other: at 8192 tokens of 32 + 8
// heads four in flight took 37.8 us, one 34.7 us, for more waves fit a CU.
template <typename E, int LPR, bool PAIRS, bool PAST>
__device__ inline void turn_heads(const Turn<LPR, PAIRS>& turn,
                                  const FmaRope& r, const FmaRows& in,
                                  long long base, typename E::raw* out, int h0,
                                  int h1, int hd, int d0, bool out_vec,
                                  bool zero, float* scratch) {
  const typename E::raw* src = static_cast<const typename E::raw*>(in.p) + base;
  for (int h = h0; h < h1; ++h) {
    float x[8];
    load8<E>(src + h * in.sh, d0, hd, in.vec != 0, x);
    turn.run(x, r, hd, d0, scratch);
    if (zero) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.0f;
    }
    store8<E, PAST>(out + static_cast<long long>(h) * hd, d0, hd, out_vec, x);
  }
}

// Which token and which of its items a row of lanes takes: the rows of one
// wave have the same item of neighbouring tokens, so they end together.
template <int LPR>
__device__ inline long long token_of(long long unit, int items, int* item) {
  constexpr int SIDE = 64 / LPR;
  const long long rest = unit / SIDE;
  const long long group = rest / items;
  *item = static_cast<int>(rest - group * items);
  return group * SIDE + unit % SIDE;
}

// A row of LPR lanes takes `per` heads of one token.
template <typename E, int LPR, bool PAIRS, bool PAST>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(
    FmaRows q, FmaRows k, void* qo, void* ko, int B, int T, int q_heads,
    int kv_heads, int hd, FmaRope r, FmaPos pos, int per, int q_items,
    int items) {
  __shared__ float scratch[256 * 8];
  const long long unit =
      static_cast<long long>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
  const int d0 = (threadIdx.x % LPR) * 8;
  int item;
  const long long bt = token_of<LPR>(unit, items, &item);
  if (bt >= static_cast<long long>(B) * T) return;
  const int b = static_cast<int>(bt / T), t = static_cast<int>(bt - 1LL * b * T);
  const bool is_q = item < q_items;
  const int heads = is_q ? q_heads : kv_heads;
  const int h0 = (is_q ? item : item - q_items) * per;
  const int h1 = min(h0 + per, heads);
  const FmaRows in = is_q ? q : k;
  typename E::raw* out =
      static_cast<typename E::raw*>(is_q ? qo : ko) + bt * heads * hd;
  Turn<LPR, PAIRS> turn;
  turn.at(r, pos_of(pos, b, t), d0);
  turn.template weights<E>(is_q ? r.qw : r.kw, d0, hd, r.w_vec != 0);
  turn_heads<E, LPR, PAIRS, PAST>(turn, r, in, b * in.sb + t * in.st, out, h0,
                                  h1, hd, d0, hd % 8 == 0, false,
                                  scratch + (threadIdx.x / LPR) * LPR * 8);
}

// ---------------------------------------------------------------------------
// Cache geometry

// Place of value (token, d) in a block of K: the A operand of
// v_mfma_f32_16x16x32 for 16 tokens by 32 values has lane 16 g + row hold
// row's values 8 g .. 8 g + 7; the two halves of the block lie side by side.
__device__ inline int kidx(int tok, int d) {
  return (((d >> 5) * 64 + ((d >> 3) & 3) * 16 + (tok & 15)) * 2 +
          (tok >> 4)) * 8 + (d & 7);
}
// Of V: the A operand of V^T, 16 values by 32 tokens. The scores come out of
// the first product with lane 16 g + row holding tokens 4 g .. 4 g + 3 of
// each half, so the k index 8 g + 4 half + r of the second product stands
// for token 16 half + 4 g + r, and the weights need no move between lanes.
__device__ inline int vidx(int tok, int d) {
  return (((d >> 5) * 64 + ((tok >> 2) & 3) * 16 + (d & 15)) * 2 +
          ((d >> 4) & 1)) * 8 + (tok >> 4) * 4 + (tok & 3);
}

struct Span {
  int start, count, end;
};
__device__ inline Span span_of(const FmaKv8Span& s, int b, int max_seq) {
  Span o;
  o.start = s.start != nullptr ? s.start[b] : s.start_i;
  int n = s.counts != nullptr ? s.counts[b] : s.T;
  n = min(n, s.T);
  if (o.start < 0 || o.start > max_seq) n = 0;
  n = min(n, max_seq - max(o.start, 0));
  o.count = max(n, 0);
  if (o.count == 0) o.start = min(max(o.start, 0), max_seq);
  o.end = o.start + o.count;
  return o;
}

// ---------------------------------------------------------------------------
// Store. One workgroup takes one block of 32 tokens of one kv head: new
// tokens go through LDS (normed, turned and rounded to 16 bits where asked),
// a block whose last token is among them is coded, and the new tokens of the
// last two blocks are also kept raw. Codes are made from the 16-bit values
// only, so they do not depend on how tokens were spread over calls.
//
// Bound by memory for prompts: 8192 tokens of 64 + 8 heads of 128 normed,
// turned and stored in int8 (319 MB) take about 68 us, 4.7 TB/s; the store of
// the 8 heads alone (50 MB) 14.5 us, where a block's wait for its maximum
// shows. One token is a launch, 3.0 us in a graph, and 5.5 us where it
// completes a block: position, values and codes are three trips to memory.

// 16 values -> 16 codes. WILD: they may be NaN, then 0, or infinite, then the
// block's largest value.
template <typename E, bool FP8, bool WILD>
__device__ inline u32x4 encode16(const uint16_t (&u)[16], float amax,
                                 float mul) {
#pragma clang fp contract(off)
  const float top = amax * mul;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float f = E::to_f(u[i]);
    x[i] = f * mul;
    if (WILD) x[i] = f == f ? fminf(fmaxf(x[i], -top), top) : 0.0f;
  }
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FP8) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w, true);
      o[i] = static_cast<uint32_t>(w);
    } else {
      // behind 1.5 * 2^23 a sum is rounded to a whole number, ties to even,
      // and its low byte is that number's; the product is rounded before
      uint32_t n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        n[j] = __float_as_uint(x[4 * i + j] + (12582912.0f + 128.0f));
      const uint32_t a = __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0400u);
      const uint32_t c = __builtin_amdgcn_perm(n[3], n[2], 0x04000c0cu);
      o[i] = a | c;
    }
  }
  return o;
}

// Scale of a block whose largest finite magnitude is amax, and what values
// are multiplied with before they are rounded. fp8: the smallest power of two
// that brings amax to 448 or less (scaling is then exact); int8: amax / 127.
template <bool FP8>
__device__ inline void scale_of(float amax, float* scale, float* mul) {
  const float a = fmaxf(amax, kMinAmax);
  if constexpr (FP8) {
    const uint32_t bits = __float_as_uint(a);
    // a = m 2^e: 448 = 1.75 * 2^8
    const int e = static_cast<int>(bits >> 23) - 127 - 8 +
                  ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    *scale = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    *mul = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  } else {
    *scale = a / 127.0f;
    *mul = 127.0f / a;
  }
}

// Which workgroups store blocks and which turn queries: 32 and then their
// share of the others in turn, so that the loads of both are under way
// together. 8192 tokens of 64 + 8 heads: 71.3 us, blocks first 79.6 us,
// queries first 84 us, one by one 88 us.
struct Share {
  bool block;
  int n;
};
__device__ inline Share share(int i, int blocks, int all) {
  const int turns = all > blocks ? blocks / 32 : 0;
  if (turns > 0) {
    const int span = 32 + (all - blocks) / turns;
    const int turn = i / span, at = i - turn * span;
    if (turn < turns)
      return at < 32 ? Share{true, turn * 32 + at}
                     : Share{false, turn * (span - 32) + at - 32};
    const int rest = i - turns * span;
    const int left = blocks - 32 * turns;
    return rest < left ? Share{true, 32 * turns + rest}
                       : Share{false, turns * (span - 32) + rest - left};
  }
  return i < blocks ? Share{true, i} : Share{false, i - blocks};
}

template <typename E, int LPR, bool PAIRS, bool FP8, bool PAST>
__global__ __launch_bounds__(256, LPR == 32 ? 3
                                            : PAIRS ? 6
                                                    : 4) void kv8_append_kernel(
    FmaKv8Layer c, FmaKv8Span sp, FmaRows q, FmaRows k, FmaRows v, void* qo,
    int q_heads, FmaRope r, int blocks, int kv_groups, int per, int q_items) {
  constexpr int MAXD = LPR * 8;
  constexpr int PITCH = MAXD + 8;
  __shared__ alignas(16) uint16_t tile[2][BLK][PITCH];
  __shared__ float scratch[256 * 8];
  __shared__ uint32_t s_max[2][4];
  const int tid = threadIdx.x;
  const int row = tid / LPR, d0 = (tid % LPR) * 8;
  constexpr int ROWS = 256 / LPR;
  float* const my_scratch = scratch + row * LPR * 8;
  const int hd = c.hd;

  const Share share_of = share(blockIdx.x, kv_groups, gridDim.x);
  if (!share_of.block) {
    int item;
    const long long bt = token_of<LPR>(
        static_cast<long long>(share_of.n) * ROWS + row, q_items, &item);
    if (bt >= static_cast<long long>(c.batch) * sp.T) return;
    const int b = static_cast<int>(bt / sp.T);
    const int t = static_cast<int>(bt - 1LL * b * sp.T);
    const Span s = span_of(sp, b, c.max_seq);
    Turn<LPR, PAIRS> turn;
    turn.at(r, s.start + t < c.max_seq ? s.start + t : 0, d0);
    turn.template weights<E>(r.qw, d0, hd, r.w_vec != 0);
    turn_heads<E, LPR, PAIRS, PAST>(
        turn, r, q, b * q.sb + t * q.st,
        static_cast<uint16_t*>(qo) + bt * q_heads * hd, item * per,
        min((item + 1) * per, q_heads), hd, d0, hd % 8 == 0, t >= s.count,
        my_scratch);
    return;
  }

  // the heads of a block next to each other: their rows are
  const int h = share_of.n % c.kv_heads;
  const int bj = share_of.n / c.kv_heads;
  const int b = bj / blocks, j = bj - b * blocks;
  const int bh = b * c.kv_heads + h;
  const Span s = span_of(sp, b, c.max_seq);
  const int b0 = s.start / BLK, blk = b0 + j;
  if (s.count == 0 || blk * BLK >= s.end) return;
  const int open = s.end / BLK;  // the block that is not complete
  const bool joins = s.start % BLK != 0;

  uint16_t* const tail = static_cast<uint16_t*>(c.tail);
  auto tail_at = [&](int which, int block) {
    return tail + which * c.tail_v +
           (static_cast<long long>(bh) * 2 + (block & 1)) * BLK * c.hdp;
  };

  // largest magnitudes, as bits; what is not finite is the largest
  u16x8 most[2] = {{0, 0, 0, 0, 0, 0, 0, 0}, {0, 0, 0, 0, 0, 0, 0, 0}};
  auto note = [&](int w, u16x8 u) {
    most[w] = __builtin_elementwise_max(most[w],
                                        u & static_cast<uint16_t>(0x7fff));
  };
  // new tokens [lo, hi) of a block: on their way, and then into LDS
  const bool as_is = r.table == 0 && r.kw == nullptr;
  constexpr int TURNS = BLK / ROWS;
  u16x8 x[TURNS], y[TURNS];
  auto fetch = [&](int block, int lo, int hi) {
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const int i = n * ROWS + row, t = block * BLK + i - s.start;
      if (block * BLK + i >= lo && block * BLK + i < hi) {
        x[n] = load_raw(static_cast<const uint16_t*>(k.p) + b * k.sb +
                            t * k.st + h * k.sh, d0, hd, k.vec != 0);
        y[n] = load_raw(static_cast<const uint16_t*>(v.p) + b * v.sb +
                            t * v.st + h * v.sh, d0, hd, v.vec != 0);
      }
    }
  };
  auto finish = [&](int block, int lo, int hi) {
    Turn<LPR, PAIRS> turn;
    turn.template weights<E>(r.kw, d0, hd, r.w_vec != 0);
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const int i = n * ROWS + row;
      if (block * BLK + i >= lo && block * BLK + i < hi) {
        if (!as_is) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = E::to_f(x[n][e]);
          turn.at(r, block * BLK + i, d0);
          turn.run(f, r, hd, d0, my_scratch);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[n][e] = d0 + e < hd ? E::from_f(f[e]) : 0;
        }
        note(0, x[n]);
        note(1, y[n]);
        *reinterpret_cast<u16x8*>(&tile[0][i][d0]) = x[n];
        *reinterpret_cast<u16x8*>(&tile[1][i][d0]) = y[n];
      }
    }
  };
  // tokens [lo, hi) of a block from LDS to its raw slot
  auto keep = [&](int block, int lo, int hi) {
    uint16_t* const kt = tail_at(0, block);
    uint16_t* const vt = tail_at(1, block);
    for (int i = lo - block * BLK + row; i < hi - block * BLK; i += ROWS) {
      if (d0 < c.hdp) {
        *reinterpret_cast<u16x8*>(kt + kidx(i, d0)) =
            *reinterpret_cast<const u16x8*>(&tile[0][i][d0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) vt[vidx(i, d0 + e)] = tile[1][i][d0 + e];
      }
    }
  };

  const int lo = max(s.start, blk * BLK), hi = min(s.end, (blk + 1) * BLK);
  fetch(blk, lo, hi);
  const bool complete = hi == (blk + 1) * BLK;
  if (complete && lo > blk * BLK) {
    // meanwhile the block's earlier tokens, eight values that lie together at
    // a time: of one token, or of eight
    const int old = lo - blk * BLK;
    const uint16_t* const kt = tail_at(0, blk);
    const uint16_t* const vt = tail_at(1, blk);
    for (int u = tid; u < c.hdp * 4; u += 256) {
      const u16x8 x = *reinterpret_cast<const u16x8*>(kt + u * 8);
      u16x8 y = *reinterpret_cast<const u16x8*>(vt + u * 8);
      const int e = u & 1, l = (u >> 1) & 63, chunk = u >> 7;
      const int g = l >> 4, n = l & 15;
      if (16 * e + n < old) {
        note(0, x);
        *reinterpret_cast<u16x8*>(&tile[0][16 * e + n][32 * chunk + 8 * g]) = x;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tok = 16 * (i >> 2) + 4 * g + (i & 3);
        if (tok < old)
          tile[1][tok][32 * chunk + 16 * e + n] = y[i];
        else
          y[i] = 0;
      }
      note(1, y);
    }
  }
  finish(blk, lo, hi);
  uint32_t top[2] = {0, 0};
  auto share = [&] {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      top[0] = max(top[0], static_cast<uint32_t>(__shfl_xor(top[0], o)));
      top[1] = max(top[1], static_cast<uint32_t>(__shfl_xor(top[1], o)));
    }
    if ((tid & 63) == 0) {
      s_max[0][tid >> 6] = top[0];
      s_max[1][tid >> 6] = top[1];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w)
      top[w] = max(max(s_max[w][0], s_max[w][1]),
                   max(s_max[w][2], s_max[w][3]));
  };
  if (complete) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        top[w] = max(top[w], static_cast<uint32_t>(most[w][e]));
    share();
  } else {
    __syncthreads();
  }

  if (complete) {
    // NaN or infinities: once more, over what is finite
    const bool wild = top[0] >= E::kInf || top[1] >= E::kInf;
    if (wild) {
      __syncthreads();
      top[0] = top[1] = 0;
      for (int i = tid; i < BLK * LPR; i += 256)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t m = tile[w][i / LPR][i % LPR * 8 + e] & 0x7fffu;
            if (i % LPR * 8 < c.hdp && m < E::kInf) top[w] = max(top[w], m);
          }
      share();
    }
    const int units = c.hdp * 2;  // of 16 values, for each of K and V
    float amax[2], mul[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      amax[w] = E::to_f(static_cast<uint16_t>(top[w]));
      float scale;
      scale_of<FP8>(amax[w], &scale, &mul[w]);
      if (tid == w)
        c.scales[w * c.scales_v + static_cast<long long>(bh) * c.nblk + blk] =
            scale;
    }
    const long long at =
        (static_cast<long long>(bh) * c.nblk + blk) * BLK * c.hdp;
    for (int i = tid; i < 2 * units; i += 256) {
      const int w = i >= units;
      const int u = i - w * units;
      const int l = u & 63, chunk = u >> 6, g = l >> 4, n = l & 15;
      uint16_t x[16];
      if (w == 0) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const u16x8 t8 = *reinterpret_cast<const u16x8*>(
              &tile[0][16 * a + n][32 * chunk + 8 * g]);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[8 * a + e] = t8[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[e] = tile[1][16 * ((e >> 2) & 1) + 4 * g + (e & 3)]
                     [32 * chunk + 16 * (e >> 3) + n];
      }
      *reinterpret_cast<u32x4*>(c.codes + w * c.codes_v + at + u * 16) =
          wild ? encode16<E, FP8, true>(x, amax[w], mul[w])
               : encode16<E, FP8, false>(x, amax[w], mul[w]);
    }
  }

  // A later block of this call may have the slot that this one's earlier
  // tokens were read from; then it is written here, after that read.
  if (blk >= open - 1 && !(joins && blk != b0 && (blk & 1) == (b0 & 1)))
    keep(blk, lo, hi);
  if (joins && blk == b0) {
    for (int other = max(open - 1, b0 + 1); other <= open; ++other) {
      if ((other & 1) == (b0 & 1) && other * BLK < s.end) {
        const int ohi = min(s.end, (other + 1) * BLK);
        __syncthreads();
        fetch(other, other * BLK, ohi);
        finish(other, other * BLK, ohi);
        __syncthreads();
        keep(other, other * BLK, ohi);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Reading back: one workgroup a block of one kv head, through LDS because a
// token's values do not lie together in V.

template <int NS, typename E, bool FP8, bool PAST>
__global__ __launch_bounds__(256) void kv8_read_kernel(
    FmaKv8Layer c, const int* start, int start_i, const int* length,
    int length_i, int n, uint16_t* ko, uint16_t* vo, int blocks) {
  constexpr int HDP = NS * 32;
  __shared__ alignas(16) uint16_t tile[BLK][HDP + 8];
  const int j = blockIdx.x % blocks;
  const int bh = blockIdx.x / blocks;
  const int b = bh / c.kv_heads, h = bh - b * c.kv_heads;
  // behind max_seq all is zero
  const int s0 = min(max(start != nullptr ? start[b] : start_i, 0), c.max_seq);
  int len = length != nullptr ? length[b] : length_i;
  len = min(max(len, 0), c.max_seq);
  const int blk = s0 / BLK + j;
  const int lo = max(s0, blk * BLK);
  const int hi = static_cast<int>(
      min(static_cast<long long>(s0) + n, (blk + 1LL) * BLK));
  if (hi <= lo) return;
  const int which = blockIdx.y;
  uint16_t* const out = which ? vo : ko;
  const bool any = blk * BLK < len;  // then blk < nblk
  if (any && blk < len / BLK) {
    const float scale = c.scales[which * c.scales_v +
                                 static_cast<long long>(bh) * c.nblk + blk];
    const unsigned char* const at =
        c.codes + which * c.codes_v +
        (static_cast<long long>(bh) * c.nblk + blk) * BLK * HDP;
#pragma unroll
    for (int u = threadIdx.x; u < HDP * 2; u += 256) {
      const int l = u & 63, chunk = u >> 6, g = l >> 4, m = l & 15;
      const u32x4 w = *reinterpret_cast<const u32x4*>(at + u * 16);
      uint16_t x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t byte = (w[e >> 2] >> (8 * (e & 3))) & 255u;
        float f;
        if constexpr (FP8)
          f = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte), 0);
        else
          f = static_cast<float>(static_cast<int>(byte) - 128);
        // a code may stand for a little more than the type's largest
        x[e] = E::from_f(fminf(fmaxf(f * scale, -E::kMost), E::kMost));
      }
      if (which) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          tile[16 * ((e >> 2) & 1) + 4 * g + (e & 3)]
              [32 * chunk + 16 * (e >> 3) + m] = x[e];
      } else {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          u16x8 v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = x[8 * a + e];
          *reinterpret_cast<u16x8*>(&tile[16 * a + m][32 * chunk + 8 * g]) = v;
        }
      }
    }
  } else if (any) {
    const uint16_t* const t =
        static_cast<const uint16_t*>(c.tail) + which * c.tail_v +
        (static_cast<long long>(bh) * 2 + (blk & 1)) * BLK * HDP;
#pragma unroll
    for (int u = threadIdx.x; u < HDP * 4; u += 256) {
      // eight values that lie together: of one token, or of eight
      const u16x8 v = *reinterpret_cast<const u16x8*>(t + u * 8);
      const int e = u & 1, l = (u >> 1) & 63, chunk = u >> 7;
      const int g = l >> 4, m = l & 15;
      if (which) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          tile[16 * (i >> 2) + 4 * g + (i & 3)][32 * chunk + 16 * e + m] = v[i];
      } else {
        *reinterpret_cast<u16x8*>(&tile[16 * e + m][32 * chunk + 8 * g]) = v;
      }
    }
  }
  __syncthreads();
  const bool vec = c.hd % 8 == 0;
  for (int u = threadIdx.x; u < (hi - lo) * NS * 4; u += 256) {
    const int p = lo + u / (NS * 4), d = u % (NS * 4) * 8;
    if (d >= c.hd) continue;
    uint16_t* const o =
        out + ((static_cast<long long>(b) * n + (p - s0)) * c.kv_heads + h) *
                  c.hd + d;
    u16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (p < len) v = *reinterpret_cast<const u16x8*>(&tile[p - blk * BLK][d]);
    if (vec) {
      put<PAST>(o, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d + i < c.hd) o[i] = v[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Attention. Query rows of one kv head (row = t * group + head) are taken 16
// at a time; S^T = K Q^T puts a row's scores into lanes 16 g + row, so the
// softmax is four lanes wide and O^T = V^T P^T takes P as it stands.
//
// K and V are made fp16 on the way into the matrix unit: e4m3 and int8 fit
// exactly. A query row is scaled by a power of two to fit fp16, exactly but
// for values 2^24 below the row's largest. The weights go in as fp16. The
// kernel for few rows waits for memory and has room for two parts of each, 20
// bits: what comes out is the plain form's but for fp32 rounding (131000 tokens
// of 4 kv heads 28.3 against 27.9 us with one part, 12 tokens behind 4000 12.1
// against 11.8 us). The one for many rows takes one, half a step of which is
// 2^-11 of a weight: against 2^-8 of a bf16 result, and as much as an fp16
// result's own where a row has no more than a few tokens for it to even out
// over. Two would cost it a third (2048 tokens behind 6144: 575 against 428
// us). So that this holds for small weights too, a row's largest stands at
// 2^8 or more (int8: 2^7): down to 2^-22 (2^-21) of the largest a weight has
// all of these bits, and below it is off by at most 2^-33 (2^-32) of the
// largest, twice that where it is cut off.
// With the largest at 1, 16384 tokens of 2^-26 beside one that holds the row,
// which first tokens of real models do, all came out as zero.
// A block's K scale multiplies its scores; its V scale relative to a running
// reference goes into V's conversion (fp8: a power of two, exact) or the
// weights (int8).

__device__ inline h8 decode8(uint32_t lo, uint32_t hi, float scale, bool fp8) {
  h2 a, b, cc, d;
  if (fp8) {
    a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true);
    cc = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false);
    d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true);
  } else {
    // 0x6400 | u is 1024 + u in fp16; less 1024 + 128 it is the code
    const h2 off = {static_cast<_Float16>(-1152.0f),
                    static_cast<_Float16>(-1152.0f)};
    const uint32_t one = 0x64646464u;
    a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one, lo, 0x04010400u)) + off;
    b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one, lo, 0x04030402u)) + off;
    cc = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one, hi, 0x04010400u)) + off;
    d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(one, hi, 0x04030402u)) + off;
  }
  return h8{a[0], a[1], b[0], b[1], cc[0], cc[1], d[0], d[1]};
}

struct AttnArgs {
  FmaKv8Layer c;
  FmaKv8Span sp;
  FmaRows q;
  void* out;
  float* partials;  // [rows, splits, HDP]: a part's own outputs
  float* stats;     // [rows, splits, 2]: reference and sum
  float scale;  // of the scores, its magnitude times log2(e)
  int negative;
  int q_heads, group, rows, tiles, splits;
};

// 16-bit values that are not finite, as finite ones: a weight of zero times
// them has to be zero.
template <typename E>
__device__ inline uint16_t tame(uint16_t u) {
  const uint32_t m = u & 0x7fffu;
  if (m < E::kInf) return u;
  return m > E::kInf ? 0
                     : static_cast<uint16_t>((u & 0x8000u) | E::kMaxFinite);
}

template <typename E>
__device__ inline f32x4 mfma16(u16x8 a, u16x8 b, f32x4 acc) {
  if constexpr (E::kInf == 0x7f80)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), acc, 0, 0, 0);
}

// Maximum over the four lanes 16 g + row that hold a row.
__device__ inline float row_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// Blocks whose largest V is under about 2^-99 (zeros): they count as nothing
// beside others.
constexpr uint32_t kNothing = (127u - 106u) << 23;

// Whether V's scales of blocks [lo, hi) lie within 2^16 of each other, the same
// in all lanes. A wave looks at all of its part's before it starts (asked
// block by block, the kernel for many rows took 4% longer): those of the first
// 64 blocks are asked for ahead of the codes, and one vote says whether all are
// within 2^8 of the first, as any model's are; only then minima and maxima.
struct Scales {
  const float* at;
  int lo, hi, lane;
  uint32_t first, mine;
  __device__ Scales(const float* vsc, int lo_, int hi_, int lane_)
      : at(vsc), lo(lo_), hi(hi_), lane(lane_) {
    first = mine = 0;
    if (lo < hi) {
      first = __float_as_uint(at[lo]);
      mine = __float_as_uint(at[min(lo + lane, hi - 1)]);
    }
  }
  __device__ bool near() const {
    constexpr uint32_t kSide = 8u << 23;
    bool odd = first < kNothing;
    uint32_t u = mine;
    for (int i = lo; i < hi; i += 64) {
      if (i > lo) u = __float_as_uint(at[min(i + lane, hi - 1)]);
      odd |= u >= kNothing && u - first + kSide > 2 * kSide;
    }
    if (__builtin_expect(!__any(odd), 1)) return true;
    uint32_t least = 0x7f800000u, most = 0;
    for (int i = lo + lane; i < hi; i += 64) {
      u = __float_as_uint(at[i]);
      if (u >= kNothing) {
        least = min(least, u);
        most = max(most, u);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      least = min(least, static_cast<uint32_t>(__shfl_xor(least, o)));
      most = max(most, static_cast<uint32_t>(__shfl_xor(most, o)));
    }
    return __builtin_amdgcn_readfirstlane(most == 0 ||
                                          most - least <= 2 * kSide);
  }
};

// The running reference of V's scales, of which a wave's outputs are
// multiples. It moves where fp16 has no room for the ratio to it (beside the
// weights, int8, there is room for a ratio of 2), and so follows blocks that
// some rows, or all, give no weight, or do not see. Within 2^16 that loses
// nothing; where scales lie further apart far_steps does without it.
template <bool FP8>
struct ScaleRef {
  static constexpr uint32_t kUp = FP8 ? 6 : 1;
  float ref = 0.0f, inv = 0.0f;
  // a difference of bits is one of exponents, to a part of one
  __device__ bool far(float scale) const {
    return static_cast<uint32_t>(__float_as_int(scale) - __float_as_int(ref) +
                                 (6 << 23)) > ((6 + kUp) << 23);
  }
  // moves it where need be; returns what to multiply outputs with
  __device__ float follow(float scale) {
    if (!far(scale) || (ref != 0.0f && __float_as_uint(scale) < kNothing))
      return 1.0f;
    const float f = ref != 0.0f ? ref / scale : 1.0f;
    ref = scale;
    inv = 1.0f / scale;
    return f;
  }
  // scale / ref; between powers of two it is a difference of exponents
  __device__ float ratio(float scale) const {
    if constexpr (FP8)
      return __int_as_float(max(
          __float_as_int(scale) - __float_as_int(ref) + 0x3f800000, 0x800000));
    else
      return scale * inv;
  }
};

// No score seen yet. Finite, so that a row that sees nothing needs no case of
// its own: its weights are exp2(-inf) and its factors multiply zeros.
constexpr float kNone = -3e38f;

// One wave's softmax and output state for 16 query rows. The reference stands
// LEAD (log2) below the largest score that it was taken from, and moves when
// one passes it by MOST: weights go up to 2^15, times 2 where V's ratio is
// beside them.
template <int NS, bool FP8>
struct RowState {
  static constexpr float LEAD = FP8 ? 8.0f : 7.0f, MOST = LEAD + 7.0f;
  f32x4 o[2 * NS];  // O^T in units of vref: value 16 n + 4 g + reg, row l % 16
  float m, l;       // running reference and this lane's share of the sum
  __device__ void clear() {
#pragma unroll
    for (int n = 0; n < 2 * NS; ++n) o[n] = f32x4{0, 0, 0, 0};
    m = kNone;
    l = 0.0f;
  }
  __device__ void times(float f) {
#pragma unroll
    for (int n = 0; n < 2 * NS; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[n][r] *= f;
  }
  __device__ void refer(float top, float more) {
    top = row_max(top);
    const float next = top > m + MOST ? top - LEAD : m;
    const float g = exp2f(m - next);
    m = next;
    l *= g;
    times(g * more);
  }
};

// x: products of NE blocks with NR times 16 rows; f > 0: what makes them log2
// scores. A row's reference moves only when a score has grown by 2^7, which
// fp16 weights and fp32 sums have room for: the outputs are rarely rescaled,
// and while no lane asks for it, no value has to cross lanes.
// more: what the outputs are to be multiplied with in any case.
template <int NR, int NE, typename RS>
__device__ inline void settle(const f32x4 (&x)[NE][NR][2],
                              const float (&f)[NE][NR], RS (&st)[NR],
                              float more) {
  float top[NR];
  bool grows = false;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      // v_maximum3: NaN comes through and moves nothing
      float y = __builtin_elementwise_maximum(x[e][r][0][0], x[e][r][0][1]);
#pragma unroll
      for (int i = 2; i < 8; ++i)
        y = __builtin_elementwise_maximum(y, x[e][r][i >> 2][i & 3]);
      y *= f[e][r];
      top[r] = e == 0 ? y : __builtin_elementwise_maximum(top[r], y);
    }
    grows |= top[r] > st[r].m + RS::MOST;
  }
  if (__any(grows) || more != 1.0f) {
#pragma unroll
    for (int r = 0; r < NR; ++r) st[r].refer(top[r], more);
  }
}
// x becomes the weights; their sum is advanced where SUM.
template <bool SUM, typename RS>
__device__ inline void weigh(f32x4 (&x)[2], float f, RS& st) {
  float sum = 0.0f;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[a][i] = __builtin_amdgcn_exp2f(fmaf(x[a][i], f, -st.m));
      if (SUM) sum += x[a][i];
    }
  if (SUM) st.l += sum;
}
// left: how many of the lane's tokens on are seen
__device__ inline void mask(f32x4 (&x)[2], int left) {
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (16 * a + i >= left) x[a][i] = -INFINITY;
}
// log2 scores of a block: K's scale times the row's factor, kept off zero and
// infinity, which would make NaN of what is masked or zero
__device__ inline float factor(float kscale, float qscale) {
  return fminf(fmaxf(kscale * qscale, 1.2e-38f), 3e38f);
}

template <bool FP8>
__device__ inline h8 weights16(const f32x4 (&x)[2], float ratio) {
  h8 p;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[4 * a + i] = static_cast<_Float16>(FP8 ? x[a][i] : x[a][i] * ratio);
  return p;
}

// The weights in two fp16 parts, 20 bits of them: both cut off, which is one
// instruction for two, for the second has what the first leaves.
template <bool FP8>
__device__ inline void weights32(const f32x4 (&x)[2], float ratio, h8* p,
                                 h8* rest) {
  u32x4 hi, lo;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[j] = x[i >> 1][2 * (i & 1) + j];
      if (!FP8) w[j] *= ratio;
    }
    const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(w[0], w[1]));
    hi[i] = __builtin_bit_cast(uint32_t, h);
    lo[i] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_pkrtz(w[0] - static_cast<float>(h[0]),
                                             w[1] - static_cast<float>(h[1])));
  }
  *p = __builtin_bit_cast(h8, hi);
  *rest = __builtin_bit_cast(h8, lo);
}

// Where a tile of query rows reads its keys: its span, the tokens stored, the
// blocks of them held as codes, those to read, and whether the tile sees the
// incomplete one.
struct Reach {
  Span s;
  int held, full, lo, hi;
  bool tail;
};
__device__ inline Reach reach_of(const AttnArgs& A, int b, int row0, int rows,
                                 int split) {
  Reach r;
  r.s = span_of(A.sp, b, A.c.max_seq);
  const int t_first = row0 / A.group;
  const int t_last =
      min((min(row0 + rows, A.rows) - 1) / A.group, r.s.count - 1);
  const int most = t_first < r.s.count ? r.s.start + t_last + 1 : 0;
  r.held = max(A.sp.held, r.s.end);
  r.full = r.held / BLK;
  const long long nb = min(r.full, (most + BLK - 1) / BLK);
  r.lo = static_cast<int>(nb * split / A.splits);
  r.hi = static_cast<int>(nb * (split + 1) / A.splits);
  r.tail = most > r.full * BLK && split == A.splits - 1;
  return r;
}

// A query row's values 32 ks + 8 g ..: as they are, and as fp16.
template <int NS, typename E>
__device__ inline void load_query(const AttnArgs& A, const uint16_t* row,
                                  bool live, int g, u16x8 (&raw)[NS]) {
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) {
    const int d = 32 * ks + 8 * g;
    raw[ks] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (live && d < A.c.hd)  // rows are padded to 16 bytes
      raw[ks] = *reinterpret_cast<const u16x8*>(row + d);
  }
}
// Returns what makes products of codes log2 scores, but for K's scale.
template <int NS, typename E>
__device__ inline float query_fp16(const AttnArgs& A, const u16x8 (&raw)[NS],
                                   h8 (&q)[NS]) {
  float top = 0.0f;
#pragma unroll
  for (int ks = 0; ks < NS; ++ks)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(E::to_f(raw[ks][i])));
  top = row_max(top);
  // 2^-e brings the row's largest into [2^9, 2^10), or as near as 2^e is a
  // normal number: also where it is bf16's largest or smallest
  int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 9;
  e = top == 0.0f ? 0 : max(e, -126);
  const float size = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  const float mul = A.negative ? -size : size;
#pragma unroll
  for (int ks = 0; ks < NS; ++ks)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      q[ks][i] = static_cast<_Float16>(E::to_f(raw[ks][i]) * mul);
  return A.scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// Blocks blk, blk + by, .. for NR times 16 rows of a wave, where V's scales lie
// further apart than one reference serves: a row's outputs are in units of
// its own, unit[r] * kFarUnit, the largest product of a weight and a scale so
// far. So neither a block that it gives no weight nor one that it does not see
// moves them, and each block's weights are rounded against its own largest.
// Any order of magnitudes of V comes out (weights under 2^-110 are dropped);
// no real model's V gets here, and a block takes two to three times as long.
constexpr float kFarUnit = 65536.0f;
template <int NS, int NR, bool FP8>
__device__ inline void far_steps(const unsigned char* kc,
                                 const unsigned char* vc, const float* ksc,
                                 const float* vsc, int lane, int blk, int hi,
                                 int by, const int (&seen)[NR],
                                 const h8 (&q)[NR][NS],
                                 const float (&qscale)[NR],
                                 RowState<NS, FP8> (&st)[NR],
                                 float (&unit)[NR]) {
  using RS = RowState<NS, FP8>;
  constexpr float kTop = 16384.0f;  // a block's largest weight in fp16
  const int g = lane >> 4;
  for (; blk < hi; blk += by) {
    const long long at = static_cast<long long>(blk) * BLK * NS * 32 + lane * 16;
    const float kscale = ksc[blk], vscale = vsc[blk] * (1.0f / kFarUnit);
    f32x4 x[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) x[r][0] = x[r][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(kc + at + ks * 1024);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const h8 kf = decode8(w[2 * a], w[2 * a + 1], 1.0f, FP8);
#pragma unroll
        for (int r = 0; r < NR; ++r)
          x[r][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[r][ks],
                                                           x[r][a], 0, 0, 0);
      }
    }
    h8 p[NR];
    float with[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float f = factor(kscale, qscale[r]);
      mask(x[r], seen[r] - blk * BLK - 4 * g);
      float top = x[r][0][0], most = 0.0f;
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[r][i >> 2][i & 3]);
      top = row_max(top * f);
      const float next = top > st[r].m + RS::MOST ? top - RS::LEAD : st[r].m;
      const float less = exp2f(st[r].m - next);
      st[r].m = next;
      st[r].l *= less;
      unit[r] *= less;
      weigh<true>(x[r], f, st[r]);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, x[r][i >> 2][i & 3]);
      most = row_max(most);
      const bool any = most > 7.7e-34f;
      const float mine = any ? most * vscale : 0.0f;
      const float now = fmaxf(unit[r], mine);
      with[r] = now > 0.0f ? mine / now * (1.0f / kTop) : 0.0f;
      st[r].times(now > 0.0f ? unit[r] / now : 1.0f);
      unit[r] = now;
      const float to = any ? kTop / most : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        p[r][i] = static_cast<_Float16>(x[r][i >> 2][i & 3] * to);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(vc + at + i * 1024);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const h8 vf = decode8(w[2 * a], w[2 * a + 1], 1.0f, FP8);
#pragma unroll
        for (int r = 0; r < NR; ++r)
          st[r].o[2 * i + a] +=
              __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  vf, p[r], f32x4{0, 0, 0, 0}, 0, 0, 0) * with[r];
      }
    }
  }
}

// What ends a wave's part of NR times 16 rows: the incomplete block, raw, where
// it reads one, and the division by the sums. Outputs are in units of
// unit[r] * more before and whole values after; l is then the row's whole sum
// in each lane.
// They are divided before the raw values and the parts of a row come together,
// so that no sum is larger than the largest V, which may be the type's largest
// (1000 tokens of 3e38 once gave infinity). A code may stand for a little more
// than that: outputs saturate, and NaN stays.
// The raw block's weights go in as two 16-bit parts: a single bf16 would cost
// as much as the result's rounding.
template <int NS, int NR, typename E, bool FP8>
__device__ inline void conclude(const AttnArgs& A, const Reach& R, bool tail,
                                int bh, int lane,
                                const uint16_t* const (&qrow)[NR],
                                const bool (&live)[NR], const int (&seen)[NR],
                                const float (&unit)[NR], float more,
                                RowState<NS, FP8> (&st)[NR]) {
  const int g = lane >> 4;
  const uint16_t* const kt =
      static_cast<const uint16_t*>(A.c.tail) +
      (static_cast<long long>(bh) * 2 + (R.full & 1)) * BLK * NS * 32 +
      lane * 16;
  const uint16_t* const vt = kt + A.c.tail_v;
  f32x4 x[1][NR][2];
  if (tail) {
    u16x8 q[NR][NS];
    float f[1][NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      load_query<NS, E>(A, qrow[r], live[r], g, q[r]);
      x[0][r][0] = x[0][r][1] = f32x4{0, 0, 0, 0};
      f[0][r] = A.scale;
    }
#pragma unroll
    for (int ks = 0; ks < NS; ++ks)
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const u16x8 k = *reinterpret_cast<const u16x8*>(kt + ks * 1024 + a * 8);
#pragma unroll
        for (int r = 0; r < NR; ++r)
          x[0][r][a] = mfma16<E>(k, q[r][ks], x[0][r][a]);
      }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (A.negative) {
        x[0][r][0] = -x[0][r][0];
        x[0][r][1] = -x[0][r][1];
      }
      mask(x[0][r], seen[r] - R.full * BLK - 4 * g);
    }
    settle<NR, 1>(x, f, st, 1.0f);
#pragma unroll
    for (int r = 0; r < NR; ++r) weigh<true>(x[0][r], A.scale, st[r]);
  }
  float by[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float l = st[r].l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    st[r].l = l;
    by[r] = l == 0.0f ? 0.0f : 1.0f / l;  // nothing seen gives zeros
    // (by times more first: unit alone may be near fp32's largest)
    st[r].times(unit[r] * (by[r] * more) * (tail ? E::kFine : 1.0f));
  }
  if (tail) {
    u16x8 hi[NR], lo[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[0][r][i >> 2][i & 3] * by[r] * E::kFine;
        const uint16_t u = E::from_f(p);
        hi[r][i] = u;
        lo[r][i] = E::from_f(p - E::to_f(u));
      }
    const int held = R.held - R.full * BLK - 4 * g;
#pragma unroll
    for (int n = 0; n < 2 * NS; ++n) {
      u16x8 v = *reinterpret_cast<const u16x8*>(vt + (n >> 1) * 1024 +
                                                (n & 1) * 8);
      const u16x8 m = v & static_cast<uint16_t>(0x7fff);
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, static_cast<uint32_t>(m[i]));
      if (__builtin_expect(__any(most >= E::kInf), 0)) {
        // NaN or infinities, in tokens or behind them
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = 16 * (i >> 2) + (i & 3) < held ? tame<E>(v[i]) : 0;
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        st[r].o[n] = mfma16<E>(v, hi[r], st[r].o[n]);
        st[r].o[n] = mfma16<E>(v, lo[r], st[r].o[n]);
        if (E::kFine != 1.0f) st[r].o[n] *= 1.0f / E::kFine;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int n = 0; n < 2 * NS; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st[r].o[n][i] = __builtin_elementwise_maximum(
            __builtin_elementwise_minimum(st[r].o[n][i], E::kMost), -E::kMost);
}

// Four values of an output row.
template <typename E>
__device__ inline void put_row(uint16_t* row, int d, int hd, f32x4 o) {
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  u16x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = E::from_f(o[i]);
  if (hd % 4 == 0) {
    if (d < hd) *reinterpret_cast<u16x4*>(row + d) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < hd) row[d + i] = u[i];
  }
}

// Few rows: four waves share 16 rows and take the blocks of a split in turn,
// each straight from memory into the matrix unit's operands, the next block
// on its way meanwhile. Bound by memory: 32 sequences of up to 8192 tokens, 8
// kv heads (270 MB), 54 us with the join, 5.0 TB/s; 131000 tokens of 4 kv
// heads in int8 28.3 us, 4.7 TB/s. On the vector unit 8 query heads a kv head
// would need more than it has: 13 codes a clock and CU arrive at 8 TB/s.
// PAST: codes that no cache would keep until they are read again are not put
// there (270 MB: 58 us against 67 us).
template <bool PAST, typename V>
__device__ inline V get(const void* at) {
  if constexpr (PAST)
    return __builtin_nontemporal_load(static_cast<const V*>(at));
  else
    return *static_cast<const V*>(at);
}
// Workgroups a CU: as many as the registers of one part of a weight left; the
// second would take one off at widths of 64 and 96 (int8, 96: 72.7 against 68.3
// us for 32 sequences of 8192 tokens).
template <int NS, bool FP8, typename E, bool PAST>
__global__ __launch_bounds__(256, NS == 1   ? 6
                                  : NS == 2 ? (FP8 ? 5 : 4)
                                  : NS == 3 ? 4
                                  : NS == 4 ? 3
                                            : 2) void kv8_attn_few_kernel(AttnArgs A) {
  constexpr int HDP = NS * 32;
  __shared__ alignas(16) float s_o[4][16][HDP + 4];
  __shared__ float s_m[4][16], s_l[4][16];
  const FmaKv8Layer& c = A.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, n16 = lane & 15;
  const int heads = c.batch * c.kv_heads;
  const int bh = blockIdx.x % heads;
  const int rest = blockIdx.x / heads;
  const int split = rest % A.splits, tile = rest / A.splits;
  const int b = bh / c.kv_heads, h = bh - b * c.kv_heads;
  const Reach R = reach_of(A, b, tile * 16, 16, split);

  const int row = tile * 16 + n16;
  const int t = row / A.group, hq = h * A.group + (row - t * A.group);
  const bool live = row < A.rows && t < R.s.count;
  const int seen = live ? R.s.start + t + 1 : 0;  // keys of this row

  RowState<NS, FP8> state[1];
  RowState<NS, FP8>& st = state[0];
  st.clear();

  if (R.lo < R.hi || R.tail) {
    const unsigned char* const kc =
        c.codes + static_cast<long long>(bh) * c.nblk * BLK * HDP + lane * 16;
    const unsigned char* const vc = kc + c.codes_v;
    const float* const ksc = c.scales + static_cast<long long>(bh) * c.nblk;
    const float* const vsc = ksc + c.scales_v;

    ScaleRef<FP8> vs;
    u32x4 kr[NS], vr[NS];
    float k_next = 0.0f, v_next = 0.0f;
    // wide heads have no registers for the next V beside this one's
    constexpr bool AHEAD = NS <= 4;
    auto load_k = [&](int blk) {
      const long long at = static_cast<long long>(blk) * BLK * HDP;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        kr[i] = get<PAST, u32x4>(kc + at + i * 1024);
      k_next = ksc[blk];
    };
    auto load_v = [&](int blk) {
      const long long at = static_cast<long long>(blk) * BLK * HDP;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        vr[i] = get<PAST, u32x4>(vc + at + i * 1024);
      v_next = vsc[blk];
    };
    const Scales scales(vsc, R.lo, R.hi, lane);
    int blk = R.lo + wave;
    if (blk < R.hi) {
      load_k(blk);
      load_v(blk);
    }
    const uint16_t* const qrow = static_cast<const uint16_t*>(A.q.p) +
                                 b * A.q.sb + t * A.q.st + hq * A.q.sh;
    u16x8 raw[1][NS];
    h8 qs[1][NS];
    h8(&q)[NS] = qs[0];
    load_query<NS, E>(A, qrow, live, g, raw[0]);
    const float qscale = query_fp16<NS, E>(A, raw[0], q);
    const int sees[1] = {seen};
    const bool near = scales.near();
    const int end = near ? R.hi : R.lo;
    for (; blk < end; blk += 4) {
      const float kscale = k_next;
      f32x4 xs[1][1][2] = {{{{0, 0, 0, 0}, {0, 0, 0, 0}}}};
      f32x4(&x)[2] = xs[0][0];
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        x[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            decode8(kr[ks][0], kr[ks][1], 1.0f, FP8), q[ks], x[0], 0, 0, 0);
        x[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            decode8(kr[ks][2], kr[ks][3], 1.0f, FP8), q[ks], x[1], 0, 0, 0);
      }
      const float vscale = v_next;
      u32x4 v_now[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) v_now[i] = vr[i];
      if (blk + 4 < R.hi) {
        load_k(blk + 4);
        if (AHEAD) load_v(blk + 4);
      }
      const float f[1][1] = {{factor(kscale, qscale)}};
      mask(x, seen - blk * BLK - 4 * g);
      settle<1, 1>(xs, f, state, vs.follow(vscale));
      weigh<true>(x, f[0][0], st);
      const float ratio = vs.ratio(vscale);
      h8 p, rest;
      weights32<FP8>(x, ratio, &p, &rest);
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        const int a = 2 * (i & 1);
        const h8 vf = decode8(v_now[i >> 1][a], v_now[i >> 1][a + 1], ratio,
                              FP8);
        st.o[i] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p, st.o[i], 0, 0, 0);
        st.o[i] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, rest, st.o[i], 0, 0, 0);
      }
      if (!AHEAD && blk + 4 < R.hi) load_v(blk + 4);
    }
    const uint16_t* const rows[1] = {qrow};
    const bool lives[1] = {live};
    float unit[1] = {vs.ref}, more = 1.0f;
    if (__builtin_expect(!near, 0)) {
      more = kFarUnit;
      const float qscales[1] = {qscale};
      far_steps<NS, 1>(kc - lane * 16, vc - lane * 16, ksc, vsc, lane, blk,
                       R.hi, 4, sees, qs, qscales, state, unit);
    }
    conclude<NS, 1, E>(A, R, R.tail && wave == 3, bh, lane, rows, lives, sees,
                       unit, more, state);
  }

  // join the four waves
#pragma unroll
  for (int n = 0; n < 2 * NS; ++n)
    *reinterpret_cast<f32x4*>(&s_o[wave][n16][16 * n + 4 * g]) = st.o[n];
  if (g == 0) {
    s_m[wave][n16] = st.m;
    s_l[wave][n16] = st.l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * HDP; i += 256) {
    const int rr = i / (HDP / 4), d = i % (HDP / 4) * 4;
    const int orow = tile * 16 + rr;
    if (orow >= A.rows) continue;
    const float m = fmaxf(fmaxf(s_m[0][rr], s_m[1][rr]),
                          fmaxf(s_m[2][rr], s_m[3][rr]));
    float f[4], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = s_l[w][rr] * __builtin_amdgcn_exp2f(s_m[w][rr] - m);
      sum += f[w];
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w)
      o += *reinterpret_cast<const f32x4*>(&s_o[w][rr][d]) * (f[w] * by);
    const int ot = orow / A.group, oh = h * A.group + (orow - ot * A.group);
    const long long at =
        (static_cast<long long>(b) * A.sp.T + ot) * A.q_heads + oh;
    if (A.splits == 1) {
      put_row<E>(static_cast<uint16_t*>(A.out) + at * c.hd, d, c.hd, o);
    } else {
      *reinterpret_cast<f32x4*>(A.partials + (at * A.splits + split) * HDP +
                                d) = o;
      if (d == 0) {
        float* const s2 = A.stats + (at * A.splits + split) * 2;
        s2[0] = m;
        s2[1] = sum;
      }
    }
  }
}

// Many rows: each of four waves has 16 * NR rows of its own, and all take the
// same blocks, NE at a time, which go through LDS as fp16, so that each value
// is decoded once for all of them; the next ones are on their way meanwhile.
// Bound by what a SIMD can issue: for each 16 products a weight costs an
// exponential and about ten other vector operations. 2048 tokens behind 6144,
// 64/8 heads of 128: 1.04e6 cycles, which is 428 to 475 us on different cards
// once the clock is up (2.2 to 2.4 GHz, after some 50 calls), 490 to 660 us
// before (2.0 GHz): 1.12 to 1.01 PFLOP/s, where a large bf16 product reaches
// 1.25. On one card each wave decoding for itself took 511 us against 495, one
// block at a time 5% more than two, 48 or 64 rows a wave (one wave a SIMD) half
// as long again.
template <int NS, bool FP8, typename E, int NR, int NE>
__global__ __launch_bounds__(256, 2) void kv8_attn_many_kernel(AttnArgs A) {
  constexpr int HDP = NS * 32;
  constexpr int UNITS = NS * 64;  // of 16 codes in a block of K or V
  // a lane's operand of each 32 by 16 values, by lanes. At a width of 192 the
  // compiler would save registers for a third workgroup on a CU, which costs
  // more than it gives (int8, 4 x 512 tokens behind 2000: 196 us against 165
  // us); 8 KB more say that none fits.
  constexpr int ROOM = NS == 6 ? 2 : 0;
  __shared__ h8 s_k[2][NE][2 * NS + ROOM][64], s_v[2][NE][2 * NS + ROOM][64];
  const FmaKv8Layer& c = A.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, n16 = lane & 15;
  const int heads = c.batch * c.kv_heads;
  const int bh = blockIdx.x % heads;
  const int rest = blockIdx.x / heads;
  // the tiles that see most first
  const int split = rest / A.tiles, tile = A.tiles - 1 - rest % A.tiles;
  const int b = bh / c.kv_heads, h = bh - b * c.kv_heads;
  constexpr int ROWS = 64 * NR;
  const Reach R = reach_of(A, b, tile * ROWS, ROWS, split);

  RowState<NS, FP8> st[NR];
  int seen[NR];
  const uint16_t* qrow[NR];
  bool live[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    st[r].clear();
    const int row = tile * ROWS + (wave * NR + r) * 16 + n16;
    const int t = row / A.group, hq = h * A.group + (row - t * A.group);
    live[r] = row < A.rows && t < R.s.count;
    seen[r] = live[r] ? R.s.start + t + 1 : 0;
    qrow[r] = static_cast<const uint16_t*>(A.q.p) + b * A.q.sb + t * A.q.st +
              hq * A.q.sh;
  }
  // blocks that every row of the wave sees whole
  const int first = (tile * ROWS + wave * NR * 16) / A.group;
  const int last_row = min(tile * ROWS + (wave + 1) * NR * 16, A.rows) - 1;
  const bool whole_wave =
      tile * ROWS + (wave + 1) * NR * 16 <= A.rows &&
      last_row / A.group < R.s.count;
  const int clear = whole_wave ? (R.s.start + first + 1) / BLK : 0;

  float unit[NR], unit_by = 1.0f;
#pragma unroll
  for (int r = 0; r < NR; ++r) unit[r] = 0.0f;
  if (R.lo < R.hi) {
    const unsigned char* const kc =
        c.codes + static_cast<long long>(bh) * c.nblk * BLK * HDP;
    const float* const ksc = c.scales + static_cast<long long>(bh) * c.nblk;
    const float* const vsc = ksc + c.scales_v;
    constexpr int EACH = (UNITS + 255) / 256;
    const unsigned char* const vc = kc + c.codes_v;
    // NE blocks of K and V, by way of registers. What lies behind the last
    // block comes as zeros, with that block's scales. Lane e of each wave
    // holds K's scale of block e, lane NE + e V's.
    struct Staged {
      u32x4 k[NE][EACH], v[NE][EACH];
      float scale;
    };
    auto load = [&](Staged& to, int blk) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const long long at = static_cast<long long>(blk + e) * BLK * HDP;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int u = threadIdx.x + i * 256;
          to.k[e][i] = to.v[e][i] = u32x4{0, 0, 0, 0};
          if ((UNITS % 256 == 0 || u < UNITS) && blk + e < R.hi) {
            to.k[e][i] = *reinterpret_cast<const u32x4*>(kc + at + u * 16);
            to.v[e][i] = *reinterpret_cast<const u32x4*>(vc + at + u * 16);
          }
        }
      }
      if (lane < 2 * NE)
        to.scale = (lane < NE ? ksc : vsc)[min(blk + lane % NE, R.hi - 1)];
    };
    const Scales scales(vsc, R.lo, R.hi, lane);
    Staged one, two;
    one.scale = two.scale = 0.0f;
    load(one, R.lo);
    if (R.lo + NE < R.hi) load(two, R.lo + NE);
    h8 q[NR][NS];
    float qscale[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      u16x8 raw[NS];
      load_query<NS, E>(A, qrow[r], live[r], g, raw);
      qscale[r] = query_fp16<NS, E>(A, raw, q[r]);
    }
    // Where the weights are not scaled the matrix unit sums them, as one more
    // row of V^T: 16 additions less for the other. l is then the row's whole
    // sum in each lane.
    h8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<_Float16>(1.0f);
    ScaleRef<FP8> vs;
    // of the blocks in LDS: K's scale, what to multiply outputs with before
    // them, and V's scale against the reference
    float kscale[NE], more[NE], ratio[NE];
    auto lane_of = [&](float x, int i) {
      return __uint_as_float(
          __builtin_amdgcn_readlane(__float_as_uint(x), i));
    };
    auto store = [&](const Staged& from, int buf) {
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const float scale = lane_of(from.scale, NE + e);
        kscale[e] = lane_of(from.scale, e);
        more[e] = vs.follow(scale);
        ratio[e] = vs.ratio(scale);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const int u = threadIdx.x + i * 256;
          if (UNITS % 256 == 0 || u < UNITS) {
            const int n = 2 * (u >> 6), l = u & 63;
            const u32x4 a = from.k[e][i], w = from.v[e][i];
            s_k[buf][e][n][l] = decode8(a[0], a[1], 1.0f, FP8);
            s_k[buf][e][n + 1][l] = decode8(a[2], a[3], 1.0f, FP8);
            s_v[buf][e][n][l] = decode8(w[0], w[1], ratio[e], FP8);
            s_v[buf][e][n + 1][l] = decode8(w[2], w[3], ratio[e], FP8);
          }
        }
      }
    };
    const bool near = scales.near();
    store(one, 0);
    __syncthreads();
    // the blocks in LDS; `later` is filled with those after the next
    auto step = [&](int blk, int buf, Staged& later, const Staged& next) {
      if (blk + 2 * NE < R.hi) load(later, blk + 2 * NE);
      f32x4 x[NE][NR][2];
      float f[NE][NR];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          f[e][r] = factor(kscale[e], qscale[r]);
          x[e][r][0] = x[e][r][1] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const h8 kf = s_k[buf][e][2 * ks + a][lane];
#pragma unroll
            for (int r = 0; r < NR; ++r)
              x[e][r][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  kf, q[r][ks], x[e][r][a], 0, 0, 0);
          }
        }
      }
      if (blk + NE > clear || blk + NE > R.hi) {
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
          for (int r = 0; r < NR; ++r)
            mask(x[e][r],
                 blk + e < R.hi ? seen[r] - (blk + e) * BLK - 4 * g : 0);
      }
      // Of two waves on a SIMD the one that is further goes first, so that
      // they do not wait for the same unit: 443 us against 467 us.
      __builtin_amdgcn_s_setprio(1);
      settle<NR, NE>(x, f, st, more[0]);
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        if (e > 0 && more[e] != 1.0f) {
#pragma unroll
          for (int r = 0; r < NR; ++r) st[r].times(more[e]);
        }
        h8 p[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          weigh<!FP8>(x[e][r], f[e][r], st[r]);
          p[r] = weights16<FP8>(x[e][r], ratio[e]);
          if (FP8)
            st[r].l = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                ones, p[r], f32x4{st[r].l, 0, 0, 0}, 0, 0, 0)[0];
        }
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int n = 0; n < 2 * NS; ++n) {
          const h8 vf = s_v[buf][e][n][lane];
#pragma unroll
          for (int r = 0; r < NR; ++r)
            st[r].o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                vf, p[r], st[r].o[n], 0, 0, 0);
        }
      }
      if (blk + NE < R.hi) store(next, buf ^ 1);
      __builtin_amdgcn_s_setprio(0);
      __syncthreads();
    };
    if (near) {
      for (int blk = R.lo; blk < R.hi; blk += 2 * NE) {
        step(blk, 0, one, two);
        if (blk + NE < R.hi) step(blk + NE, 1, two, one);
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        unit[r] = vs.ref;
        if (FP8) st[r].l *= 0.25f;  // this lane's share again
      }
    } else {
      unit_by = kFarUnit;
      far_steps<NS, NR>(kc, vc, ksc, vsc, lane, R.lo, R.hi, 1, seen, q, qscale,
                        st, unit);
    }
  }
  conclude<NS, NR, E>(A, R, R.tail, bh, lane, qrow, live, seen, unit, unit_by,
                      st);

#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = tile * ROWS + (wave * NR + r) * 16 + n16;
    if (row >= A.rows) continue;
    const int t = row / A.group, hq = h * A.group + (row - t * A.group);
    const long long at =
        (static_cast<long long>(b) * A.sp.T + t) * A.q_heads + hq;
    if (A.splits == 1) {
      uint16_t* const out = static_cast<uint16_t*>(A.out) + at * c.hd;
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n)
        put_row<E>(out, 16 * n + 4 * g, c.hd, st[r].o[n]);
    } else {
      float* const part = A.partials + (at * A.splits + split) * HDP;
#pragma unroll
      for (int n = 0; n < 2 * NS; ++n)
        *reinterpret_cast<f32x4*>(part + 16 * n + 4 * g) = st[r].o[n];
      if (g == 0) {
        float* const s2 = A.stats + (at * A.splits + split) * 2;
        s2[0] = st[r].m;
        s2[1] = st[r].l;
      }
    }
  }
}

// Joins the splits of a row, always in the same order: one workgroup a row,
// as many splits at once as have a lane for each four values. The values are
// asked for before the weights are known.
template <int NS, typename E>
__global__ __launch_bounds__(256) void kv8_join_kernel(const float* partials,
                                                       const float* stats,
                                                       uint16_t* out,
                                                       int splits, int hd) {
  constexpr int HDP = NS * 32, LANES = HDP / 4, GROUPS = 256 / LANES;
  constexpr int TURNS = (kMaxSplits + GROUPS - 1) / GROUPS;
  __shared__ float s_w[kMaxSplits];
  __shared__ f32x4 s_o[GROUPS][LANES];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, grp = tid / LANES, lane = tid % LANES;
  const float* const p = partials + row * splits * HDP + lane * 4;
  f32x4 x[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int s = grp + i * GROUPS;
    x[i] = f32x4{0, 0, 0, 0};
    if (grp < GROUPS && s < splits)
      x[i] = *reinterpret_cast<const f32x4*>(p + static_cast<long long>(s) * HDP);
  }
  if (tid < 64) {
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = tid + 64 * i;
      const float* const st = stats + (row * splits + s) * 2;
      m[i] = s < splits ? st[0] : kNone;
      l[i] = s < splits ? st[1] : 0.0f;
    }
    float top = fmaxf(m[0], m[1]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] *= exp2f(m[i] - top);
      sum += l[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 2; ++i) s_w[tid + 64 * i] = l[i] * by;
  }
  __syncthreads();
  if (grp < GROUPS) {
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int s = grp + i * GROUPS;
      if (s < splits) {
        const float w = s_w[s];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = fmaf(x[i][r], w, o[r]);
      }
    }
    s_o[grp][lane] = o;
  }
  __syncthreads();
  for (int d = tid; d < hd; d += 256) {
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) o += s_o[i][d >> 2][d & 3];
    out[row * hd + d] = E::from_f(o);
  }
}

// The same for many rows of few splits: a row of lanes each.
template <int NS, typename E>
__global__ __launch_bounds__(256) void kv8_join_rows_kernel(
    const float* partials, const float* stats, uint16_t* out, long long rows,
    int splits, int hd) {
  constexpr int HDP = NS * 32, LANES = HDP / 4, GROUPS = 256 / LANES;
  const int grp = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
  const long long row = static_cast<long long>(blockIdx.x) * GROUPS + grp;
  if (grp >= GROUPS || row >= rows) return;
  const float* const st = stats + row * splits * 2;
  const float* const p = partials + row * splits * HDP + d;
  float top = kNone;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, st[2 * s]);
  float sum = 0.0f;
  for (int s = 0; s < splits; ++s)
    sum += __builtin_amdgcn_exp2f(st[2 * s] - top) * st[2 * s + 1];
  const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
  f32x4 o = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s)
    o += *reinterpret_cast<const f32x4*>(p + static_cast<long long>(s) * HDP) *
         (__builtin_amdgcn_exp2f(st[2 * s] - top) * st[2 * s + 1] * by);
  put_row<E>(out + row * hd, d, hd, o);
}

// Heads that a row of lanes takes: as many as leave every CU six workgroups
// of 256 threads, at most 16 (8192 tokens of 32 + 8 heads: 4 heads 38.6 us, 8
// 34.7 us, 16 31.7 us, 32 37.9 us).
int heads_each(long long rows, int heads) {
  const long long n = rows / (256 * 6 * 16);
  const int most = n < 1 ? 1 : n > 16 ? 16 : static_cast<int>(n);
  const int items = (heads + most - 1) / most;  // of like size
  return (heads + items - 1) / items;
}
// Outputs beyond the 32 MB of second-level caches are stored past them: at
// 84 MB 37.8 us against 50.7 us.
bool past_caches(long long bytes) { return bytes > (32LL << 20); }

int lanes_per_row(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }

// Workgroups for `items` rows of lanes a token, as token_of hands them out.
long long token_groups(long long tokens, int items, int hd) {
  const int rows = 256 / lanes_per_row(hd), side = 64 / lanes_per_row(hd);
  const long long units = (tokens + side - 1) / side * side * items;
  return (units + rows - 1) / rows;
}

// A launch takes fewer than 2^32 threads in x.
template <typename... P, typename... Given>
hipError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t lds,
                  hipStream_t stream, Given... given) {
  if (static_cast<long long>(grid.x) * threads > 0xffffffffLL)
    return hipErrorInvalidValue;
  return [&](P... args) {
    void* list[] = {&args...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid,
                           dim3(threads), list, lds, stream);
  }(given...);
}

}  // namespace

#define FMA_BY_TYPE(type, ...)                                 \
  if ((type) == 0) { using E = Bf16; __VA_ARGS__; }            \
  else if ((type) == 1) { using E = Fp16; __VA_ARGS__; }       \
  else { using E = Fp32; __VA_ARGS__; }
#define FMA_BY_TYPE16(bf16, ...)                               \
  if (bf16) { using E = Bf16; __VA_ARGS__; }                   \
  else { using E = Fp16; __VA_ARGS__; }
#define FMA_BY_BOOL(cond, NAME, ...)                           \
  if (cond) { constexpr bool NAME = true; __VA_ARGS__; }       \
  else { constexpr bool NAME = false; __VA_ARGS__; }
#define FMA_BY_LANES(hd, ...)                                  \
  if (lanes_per_row(hd) == 8) { constexpr int LPR = 8; __VA_ARGS__; }          \
  else if (lanes_per_row(hd) == 16) { constexpr int LPR = 16; __VA_ARGS__; }   \
  else { constexpr int LPR = 32; __VA_ARGS__; }
#define FMA_BY_WIDTH(hdp, ...)                                 \
  switch ((hdp) / 32) {                                        \
    case 1: { constexpr int NS = 1; __VA_ARGS__; } break;      \
    case 2: { constexpr int NS = 2; __VA_ARGS__; } break;      \
    case 3: { constexpr int NS = 3; __VA_ARGS__; } break;      \
    case 4: { constexpr int NS = 4; __VA_ARGS__; } break;      \
    case 6: { constexpr int NS = 6; __VA_ARGS__; } break;      \
    case 8: { constexpr int NS = 8; __VA_ARGS__; } break;      \
    default: return hipErrorInvalidValue;                      \
  }

extern "C" hipError_t fma_launch_qk_norm_rope(
    FmaRows q, FmaRows k, void* qo, void* ko, int B, int T, int q_heads,
    int kv_heads, int hd, int type, FmaRope rope, FmaPos pos,
    hipStream_t stream) {
  const long long tokens = static_cast<long long>(B) * T;
  if (tokens == 0) return hipSuccess;
  const int per = heads_each(tokens * (q_heads + kv_heads), q_heads);
  const int q_items = (q_heads + per - 1) / per;
  const int items = q_items + (kv_heads + per - 1) / per;
  const long long grid = token_groups(tokens, items, hd);
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  FMA_BY_TYPE(type, FMA_BY_LANES(hd, FMA_BY_BOOL(rope.pairs, PAIRS,
      FMA_BY_BOOL(past_caches(tokens * (q_heads + kv_heads) * hd *
                              (type == 2 ? 4 : 2)), PAST,
          return launch(qk_norm_rope_kernel<E, LPR, PAIRS, PAST>,
                        dim3(static_cast<unsigned>(grid)), 256, 0, stream, q,
                        k, qo, ko, B, T, q_heads, kv_heads, hd, rope, pos, per,
                        q_items, items)))));
}

extern "C" hipError_t fma_launch_kv8_append(FmaKv8Layer c, FmaKv8Span span,
                                            FmaRows q, FmaRows k, FmaRows v,
                                            void* qo, int q_heads,
                                            FmaRope rope, hipStream_t stream) {
  const long long tokens = static_cast<long long>(c.batch) * span.T;
  if (tokens == 0) return hipSuccess;
  int blocks = (span.T + BLK - 2) / BLK + 1;
  if (span.start == nullptr)
    blocks = (span.start_i + span.T - 1) / BLK - span.start_i / BLK + 1;
  const long long kv_groups =
      static_cast<long long>(c.batch) * c.kv_heads * blocks;
  const int per = heads_each(tokens * q_heads, q_heads > 0 ? q_heads : 1);
  const int q_items = (q_heads + per - 1) / per;
  const long long q_groups =
      q.p == nullptr ? 0 : token_groups(tokens, q_items, c.hd);
  if (kv_groups + q_groups > 0x7fffffffLL) return hipErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(kv_groups + q_groups);
  FMA_BY_TYPE16(c.bf16, FMA_BY_LANES(c.hd, FMA_BY_BOOL(rope.pairs, PAIRS,
      FMA_BY_BOOL(c.fp8, FP8,
          FMA_BY_BOOL(past_caches(tokens * q_heads * c.hd * 2), PAST,
              return launch(kv8_append_kernel<E, LPR, PAIRS, FP8, PAST>,
                            dim3(grid), 256, 0, stream, c, span, q, k, v, qo,
                            q_heads, rope, blocks, static_cast<int>(kv_groups),
                            per, q_items))))));
}

extern "C" hipError_t fma_launch_kv8_read(FmaKv8Layer c, const int* start,
                                          int start_i, const int* length,
                                          int length_i, int n, void* ko,
                                          void* vo, hipStream_t stream) {
  if (n == 0 || c.batch == 0) return hipSuccess;
  const int blocks = (n + BLK - 2) / BLK + 1;
  const long long groups = static_cast<long long>(c.batch) * c.kv_heads * blocks;
  if (groups > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(groups), 2);
  FMA_BY_TYPE16(c.bf16, FMA_BY_BOOL(c.fp8, FP8, FMA_BY_WIDTH(c.hdp,
      FMA_BY_BOOL(past_caches(4LL * n * c.batch * c.kv_heads * c.hd), PAST,
          return launch(kv8_read_kernel<NS, E, FP8, PAST>, grid, 256, 0,
                        stream, c, start, start_i, length, length_i, n,
                        static_cast<uint16_t*>(ko), static_cast<uint16_t*>(vo),
                        blocks)))));
}

namespace {
constexpr int many_nr(int ns) { return ns <= 4 ? 2 : 1; }
constexpr int many_ne(int ns) { return ns <= 4 ? 2 : 1; }
}  // namespace

extern "C" FmaKv8Plan fma_kv8_attn_plan(const FmaKv8Layer* c, int T,
                                        int q_heads, int max_len, int cus) {
  const long long rows = static_cast<long long>(T) * (q_heads / c->kv_heads);
  const long long heads = static_cast<long long>(c->batch) * c->kv_heads;
  const int nb = max_len / BLK;
  const double wide = c->hdp / 128.0;
  FmaKv8Plan plan;
  // Tiles of 16 rows read the codes once each, so up to 64 rows they are taken
  // while that is little: 8 kv heads of 128, 4000 tokens, 48 rows: 12.2 us
  // against 19.2 us for one sequence, 37.0 against 35.9 us for eight (195 MB),
  // 109 against 85 us for 32.
  const double codes = 64.0 * nb * heads * c->hdp;
  const long long few = (rows + 15) / 16;
  if (few <= 1 || (few <= 4 && few * codes * wide <= 200e6)) {
    plan.tile = 16;
    // A join costs 2.5 us, so short axes stay whole (heads of 128, 8 kv heads,
    // one sequence: 24 blocks 7.5 us whole, 7.7 us in eight; 32 blocks 8.6 and
    // 7.8 us). Then a workgroup for each CU while each has four blocks; and
    // four for each CU, for sequences of different length to even out, while
    // each has 16: eight sequences of 4095 tokens in 1 / 4 / 8 / 16 parts 30.4
    // / 17.1 / 15.0 / 17.0 us; 32 of up to 8192 in 1 / 2 / 4 / 8 / 16 parts
    // 74.0 / 61.5 / 58.1 / 60.0 / 66.4 us.
    const long long all = few * heads;
    plan.splits = 1;
    if (all > 0 && nb > (c->hdp <= 128 ? 24 : 16)) {
      const long long one = cus / all < nb / 4 ? cus / all : nb / 4;
      const long long four = 4LL * cus / all < nb / 16 ? 4LL * cus / all
                                                       : nb / 16;
      const long long most = one > four ? one : four;
      plan.splits = most < 1            ? 1
                    : most > kMaxSplits ? kMaxSplits
                                        : static_cast<int>(most);
    }
    return plan;
  }
  // Many rows: what two blocks take a workgroup alone on its CU, or two of
  // them together, with four blocks' worth to begin and end; a join, whose
  // parts are written and read at 3.5 TB/s. As measured for 298 shapes in 1 to
  // 32 parts (widths 64 to 256, 24 to 1024 tokens behind 0 to 32000, 1 to 16
  // sequences): what is chosen is on the mean 0.2% from the best, at most 9%;
  // without the beginning and the end 1.3% and 31%.
  plan.tile = 64 * many_nr(c->hdp / 32);
  const double groups =
      static_cast<double>((rows + plan.tile - 1) / plan.tile) * heads;
  const double w = wide < 1.25 ? wide : 1.25;
  const double all = static_cast<double>(c->batch) * T * q_heads;
  double best = 0.0;
  plan.splits = 1;
  for (int n = 1; n <= kMaxSplits && (n == 1 || n <= nb / 2); n *= 2) {
    const double turns = groups * n / (2.0 * cus);
    const double pair = groups * n <= cus
                            ? 0.4 + 1.3 * w
                            : (0.6 + 1.1 * w) * (turns > 1.0 ? turns : 1.0);
    const double us = (nb / (2.0 * n) + 4.0) * pair +
                      (n > 1 ? 2.0 + all * n * c->hdp * 8.0 / 3.5e6 : 0.0);
    if (n == 1 || us < best) {
      best = us;
      plan.splits = n;
    }
  }
  return plan;
}

extern "C" hipError_t fma_launch_kv8_attention(FmaKv8Layer c, FmaKv8Span span,
                                               FmaRows q, void* out,
                                               int q_heads, float scale,
                                               float* partials,
                                               FmaKv8Plan plan,
                                               hipStream_t stream) {
  if (c.batch == 0 || span.T == 0) return hipSuccess;
  AttnArgs a;
  a.c = c;
  a.sp = span;
  a.q = q;
  a.out = out;
  a.partials = partials;
  a.stats = partials + static_cast<long long>(c.batch) * span.T * q_heads *
                           plan.splits * c.hdp;
  a.scale = fmaxf(fabsf(scale) * kLog2e, 1.2e-38f);
  a.negative = scale < 0.0f;
  a.q_heads = q_heads;
  a.group = q_heads / c.kv_heads;
  const long long rows = static_cast<long long>(span.T) * a.group;
  const long long all = static_cast<long long>(c.batch) * span.T * q_heads;
  const int tile = plan.tile, splits = plan.splits;
  const long long tiles = (rows + tile - 1) / tile;
  const long long grid = tiles * c.batch * c.kv_heads * splits;
  if (rows > 0x7fffff00LL || all > 0x7fffffffLL || grid > 0x7fffffffLL)
    return hipErrorInvalidValue;
  a.rows = static_cast<int>(rows);
  a.tiles = static_cast<int>(tiles);
  a.splits = splits;
  const long long held =
      span.start == nullptr ? span.start_i + span.T : c.max_seq;
  const bool past = past_caches(2 * held * c.batch * c.kv_heads * c.hdp);
  hipError_t err = hipSuccess;
  const dim3 g(static_cast<unsigned>(grid));
  if (tile == 16) {
    FMA_BY_TYPE16(c.bf16, FMA_BY_BOOL(c.fp8, FP8, FMA_BY_WIDTH(c.hdp,
        FMA_BY_BOOL(past, PAST,
            err = launch(kv8_attn_few_kernel<NS, FP8, E, PAST>, g, 256, 0,
                         stream, a)))));
  } else {
    FMA_BY_TYPE16(c.bf16, FMA_BY_BOOL(c.fp8, FP8, FMA_BY_WIDTH(c.hdp,
        err = launch(kv8_attn_many_kernel<NS, FP8, E, many_nr(NS), many_ne(NS)>,
                     g, 256, 0, stream, a))));
  }
  if (err != hipSuccess || splits == 1) return err;
  if (all >= 2048) {
    FMA_BY_TYPE16(c.bf16, FMA_BY_WIDTH(c.hdp,
        constexpr int GROUPS = 256 / (NS * 8);
        return launch(kv8_join_rows_kernel<NS, E>,
                      dim3(static_cast<unsigned>((all + GROUPS - 1) / GROUPS)),
                      256, 0, stream, a.partials, a.stats,
                      static_cast<uint16_t*>(out), all, splits, c.hd)));
  }
  FMA_BY_TYPE16(c.bf16, FMA_BY_WIDTH(c.hdp,
      return launch(kv8_join_kernel<NS, E>, dim3(static_cast<unsigned>(all)),
                    256, 0, stream, a.partials, a.stats,
                    static_cast<uint16_t*>(out), splits, c.hd)));
}
