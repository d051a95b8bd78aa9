// Rows held in 8 bits: whole numbers q[j] = round(127 y[j] / max |y|), ties to the even one, and one fp32 scale max |y| / 127 per row, written where
// the row is made: from the RMS norm of x (+ residual), from a gated activation, or from a row as it is.  And back: q[j] * scale.
//
// The mathematics.  A norm multiplies a row by a factor f = rsqrt(mean h^2 + eps) of its own, which leaves q as it is and joins the scale, so the sum
// of squares and the largest |h w| are taken in one pass over the row and one exchange between its threads.  127 y / max |y| is formed with the reciprocal
// of max |y| (off by at most 127 * 2^-22); for elements that this leaves within 1e-4 of a tie the sign of 127 y - border max |y|, in one
// fused operation, says on which side of it they are.  bf16 rows need this: half of the largest value lies on a tie, and a row often holds it.
// The sum of squares holds for elements from 2^-45 to 2^63; rows beyond that are made again in 64 bits at the end (rows_in_64_bits).
// A row below 2^-100 (or, ahead of its factor, below 2^-120) is stored as zeros with scale 0; a row with an infinity or a NaN as zeros with scale NaN, so
// that everything made from it is NaN.
//
// What bounds it: memory.  One pass reads the inputs and writes 1 byte per element (and h, 2 or 4).  The threads of a row keep it in registers as fp32
// between the reduction and the write, and the reads of a block's next row are under way meanwhile:
//   - rows of whole groups of 16 bf16 elements that start on 32 bytes, above 512 and up to 16384 columns: a block per row, one load of 32 bytes per thread
//     and input (rows16_kernel).  16384 x 4096: norm with residual 73 us (470 MB, 6.4 TB/s), without 48 (4.2), a row as it is 38 (5.3); gated activation of
//     8192 x 11008 84 (5.4), of which 70 would be the bytes.  A norm without residual waits for its reduction: of 4096 columns it holds half of what an SM could read in that time.
//   - the others (quantize_kernel): up to 512 columns a warp per row; up to 16384 a block per row, eight elements per thread and turn; beyond that (norms with
//     residual: beyond 12288, in fp32 8192) the row is read twice.  Rows of 4095 or 11007 columns, which start anywhere: 16384 x 4095 norm with residual 200 us, a row
//     as it is 65; gated activation of 8192 x 11007 187 (floors 73, 31 and 70): one aligned load more per eight elements and a shift per word, and the registers that
//     they take leave one block per SM.  fp32 norms with residual of more than 8192 columns read twice what they could read once: 8192 x 11008 268 us, floor 181.
//   - back: 31 us for 16384 x 4096 (201 MB, 6.4 TB/s), 42 for 8192 x 11008; rows of odd widths 45 and 58.
// Few rows are bound by a launch: one row of 4096 takes 2.0 us in a graph.
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace lvb {
namespace int8_rows {

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100
constexpr float kLeast = 7.52316384526264e-37f;  // 2^-120: 127 over it is still a finite number
constexpr float kMostScale = 0x1.020406p+121f;   // times 127 it is still a finite number

enum Act : int { kSilu = 0, kGeluTanh = 1, kGelu = 2, kRelu = 3, kQuickGelu = 4 };

// x sigmoid(a x) of two numbers with the quick exponential and reciprocal, for fp32 gates as well: right to 2^-20 where |a x| is up to 8 and to 2^-23 |a x| beyond (the
// exponent's argument is rounded).  Half a step of the 8 bits is 2^-8 of the row's largest element, so an element goes to the other whole number only where it lies
// that close to the border.  With expf and a division, fp32 rows of 8192 x 11008 take 334 us instead of 233 and 65536 x 256 105 instead of 54.  An exponential
// that runs over makes the quotient 0, as it should be.
__device__ __forceinline__ F32x2 swish2(F32x2 x, float a) {
  const float k = -1.4426950408889634f * a;  // log2 e
  float e0, e1;
  f2_split(f2_mul(x, f2(k, k)), e0, e1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
  f2_split(f2_add(f2(e0, e1), f2(1.f, 1.f)), e0, e1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
  return f2_mul(x, f2(e0, e1));
}
template <int kAct>
__device__ __forceinline__ F32x2 activation2(F32x2 g) {
  if constexpr (kAct == kSilu) return swish2(g, 1.f);
  if constexpr (kAct == kQuickGelu) return swish2(g, 1.702f);
  if constexpr (kAct == kGeluTanh) {  // (1 + tanh u) / 2 = sigmoid(2 u)
    const F32x2 g2 = f2_mul(g, g), u = f2_mul(g, f2_fma(g2, f2(0.044715f, 0.044715f), f2(1.f, 1.f)));
    const float k = -1.4426950408889634f * 2.f * 0.7978845608028654f;
    float e0, e1;
    f2_split(f2_mul(u, f2(k, k)), e0, e1);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
    f2_split(f2_add(f2(e0, e1), f2(1.f, 1.f)), e0, e1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e1));
    return f2_mul(g, f2(e0, e1));
  }
  float a, b;
  f2_split(g, a, b);
  if constexpr (kAct == kGelu) return f2(0.5f * a * (1.f + erff(a * 0.7071067811865476f)), 0.5f * b * (1.f + erff(b * 0.7071067811865476f)));
  return f2(a != a ? a : fmaxf(a, 0.f), b != b ? b : fmaxf(b, 0.f));
}

// ---- eight elements of a row
// A row may start anywhere.  Where it does not start on 16 bytes, one aligned load more and a shift bring the eight elements (the neighbouring lanes'
// loads overlap in the L1); at the ends of what the caller gave, [lo, hi), they come one by one.
template <typename T>
struct Span {
  const T* p;
  long long ld;
  const char *lo, *hi;
  Span() = default;
  Span(const void* x, long long ld, long long rows, int cols)
      : p(static_cast<const T*>(x)), ld(ld), lo(static_cast<const char*>(x)), hi(reinterpret_cast<const char*>(static_cast<const T*>(x) + (rows - 1) * ld + cols)) {}
};
// The words that follow the first `bytes` (even, below 16) of u, moved to its front.
template <int kOut, int kIn>
__device__ __forceinline__ void shift_words(uint32_t (&u)[kIn], uint32_t bytes) {
  static_assert(kIn >= kOut + 4, "three words and a half may go");
  if (bytes & 8)
#pragma unroll
    for (int j = 0; j < kOut + 2; ++j) u[j] = u[j + 2];
  if (bytes & 4)
#pragma unroll
    for (int j = 0; j < kOut + 1; ++j) u[j] = u[j + 1];
  if (bytes & 2)
#pragma unroll
    for (int j = 0; j < kOut; ++j) u[j] = __funnelshift_r(u[j], u[j + 1], 16);
}
template <typename T>
struct Raw {  // eight elements as they lie in memory, and ahead of them what an aligned load brings along
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t u[kWords + 4];
  uint32_t before;  // bytes ahead of the first element
  __device__ __forceinline__ void load(const T* p, int live, const char* lo, const char* hi) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    const char* base = reinterpret_cast<const char*>(p) - off;
    const bool inside = live >= 8 && (off == 0 || (base >= lo && base + 4 * kWords + 16 <= hi));
    before = inside ? off : 0;
    if (inside) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(base) + i);
        u[4 * i] = w.x; u[4 * i + 1] = w.y; u[4 * i + 2] = w.z; u[4 * i + 3] = w.w;
      }
      if (off != 0) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(base) + kWords / 4);
        u[kWords] = w.x; u[kWords + 1] = w.y; u[kWords + 2] = w.z; u[kWords + 3] = w.w;
      }
    } else if constexpr (sizeof(T) == 2) {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = (2 * j < live ? __ldg(q + 2 * j) : 0u) | (2 * j + 1 < live ? static_cast<uint32_t>(__ldg(q + 2 * j + 1)) << 16 : 0u);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = j < live ? __float_as_uint(__ldg(p + j)) : 0u;
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {  // (not ahead of here: loads that have just been started are not waited for)
    uint32_t e[kWords + 4];
#pragma unroll
    for (int j = 0; j < kWords + 4; ++j) e[j] = u[j];
    if (before != 0) shift_words<kWords>(e, before);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(e[j] << 16);
        v[2 * j + 1] = __uint_as_float(e[j] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(e[j]);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    before = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(v[j]);
    }
  }
  __device__ __forceinline__ void put(T* p, int from, int to) const {  // elements [from, to) one by one
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= from && j < to) {
        if constexpr (sizeof(T) == 2) reinterpret_cast<unsigned short*>(p)[j] = static_cast<unsigned short>(u[j / 2] >> (16 * (j & 1)));
        else reinterpret_cast<uint32_t*>(p)[j] = u[j];
      }
  }
  // All lanes of a warp, each with the eight elements behind those of the lane before it (`live` of them exist, none where it is not positive).  Where they do not
  // start on 16 bytes, a lane writes the aligned words up to its last whole ones, the first of them with the end of what the lane before it holds.
  __device__ __forceinline__ void store(T* p, int live) const {
    const int lane = threadIdx.x & 31;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
    if (off == 0) {
      if (live >= 8) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
      } else if (live > 0) {
        put(p, 0, live);
      }
      return;
    }
    uint32_t e[kWords + 4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = __shfl_up_sync(0xffffffffu, u[kWords - 4 + j], 1);
#pragma unroll
    for (int j = 0; j < kWords; ++j) e[4 + j] = u[j];
    const int tail = static_cast<int>(off / sizeof(T));  // elements of a lane that the next lane writes, if it has eight
    if (live >= 8 && lane > 0) {
      shift_words<kWords>(e, 16 - off);
      uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<char*>(p) - off);
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) q[i] = make_uint4(e[4 * i], e[4 * i + 1], e[4 * i + 2], e[4 * i + 3]);
      if (lane == 31 || live < 16) put(p, 8 - tail, 8);
    } else if (live > 0) {
      put(p, 0, lane == 0 && live >= 16 ? 8 - tail : min(live, 8));
    }
  }
};

// ---- where a row comes from: load() starts the reads of eight of its elements, get() gives them and adds what the row's factor needs to `ss`.  kWide: it takes
// many registers; kMostHeld: the most threads whose registers hold a row (both: quantize()).  All
// lanes of a warp call get(); `live` of the elements exist (none where it is not positive), the others are zero.
template <typename T>
struct Plain {
  Span<T> x;
  using In = Raw<T>;
  static constexpr bool kSum = false, kWide = false;
  static constexpr int kMostHeld = 1024;
  __device__ __forceinline__ void load(In& in, long long row, int c, int live) const { in.load(x.p + row * x.ld + c, live, x.lo, x.hi); }
  __device__ __forceinline__ void get(const In& in, long long, int, int, float (&y)[8], F32x2&) const { in.get(y); }
  __device__ __forceinline__ float factor(float) const { return 1.f; }
};

// What a norm is made of when its rows have been added: for rows_in_64_bits().
template <typename T>
struct Normed {
  const T* rows;
  const void* w;
  long long ld;
  int w_f32;
  float w_offset, eps;
  __device__ __forceinline__ float element(long long row, int c) const { return static_cast<float>(rows[row * ld + c]); }
  __device__ __forceinline__ float weight(int c) const {
    return w == nullptr ? 1.f : w_offset + (w_f32 ? static_cast<const float*>(w)[c] : static_cast<float>(static_cast<const __nv_bfloat16*>(w)[c]));
  }
};

template <typename T, bool kResidual>
struct Norm {
  Span<T> x, r;
  T* h;  // written where there is a residual
  const void* w;
  long long ldh;
  int w_f32;
  float w_offset, eps, per_col;  // per_col: 1 / columns
  struct In {
    Raw<T> a, b;  // (without a residual the second is never loaded and takes no register)
  };
  static constexpr bool kSum = true, kWide = kResidual;
  static constexpr int kMostHeld = !kResidual ? 1024 : sizeof(T) == 2 ? 768 : 512;
  __device__ __forceinline__ void load(In& in, long long row, int c, int live) const {
    in.a.load(x.p + row * x.ld + c, live, x.lo, x.hi);
    if constexpr (kResidual) in.b.load(r.p + row * r.ld + c, live, r.lo, r.hi);
  }
  template <typename W>
  __device__ __forceinline__ void weigh(const W* p, int live, float (&y)[8]) const {
    Raw<W> raw;
    raw.load(p, live, nullptr, nullptr);
    float f[8];
    raw.get(f);
    if (w_offset != 0.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += w_offset;
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) f2_split(f2_mul(f2(y[j], y[j + 1]), f2(f[j], f[j + 1])), y[j], y[j + 1]);
  }
  __device__ __forceinline__ void get(const In& in, long long row, int c, int live, float (&y)[8], F32x2& ss) const {
    in.a.get(y);
    if constexpr (kResidual) {
      float b[8];
      in.b.get(b);
#pragma unroll
      for (int j = 0; j < 8; j += 2) f2_split(f2_add(f2(y[j], y[j + 1]), f2(b[j], b[j + 1])), y[j], y[j + 1]);
      Raw<T> sum;
      sum.set(y);
      sum.get(y);  // the sum in the rows' type is what goes on, here too
      sum.store(h + row * ldh + c, live);
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) ss = f2_fma(f2(y[j], y[j + 1]), f2(y[j], y[j + 1]), ss);
    if (w != nullptr && live > 0) {
      if (w_f32) weigh(reinterpret_cast<const float*>(w) + c, live, y);
      else weigh(reinterpret_cast<const __nv_bfloat16*>(w) + c, live, y);
    }
  }
  __device__ __forceinline__ float mean(float ss) const { return ss * per_col + eps; }
  __device__ __forceinline__ float factor(float ss) const { return rsqrtf(mean(ss)); }
  __device__ __forceinline__ Normed<T> normed(long long) const { return {kResidual ? h : x.p, w, kResidual ? ldh : x.ld, w_f32, w_offset, eps}; }
};

template <typename T, int kAct>
struct Glu {
  Span<T> g, u;
  struct In {
    Raw<T> a, b;
  };
  static constexpr bool kSum = false, kWide = sizeof(T) == 4;
  static constexpr int kMostHeld = 1024;
  __device__ __forceinline__ void load(In& in, long long row, int c, int live) const {
    in.a.load(g.p + row * g.ld + c, live, g.lo, g.hi);
    in.b.load(u.p + row * u.ld + c, live, u.lo, u.hi);
  }
  __device__ __forceinline__ void get(const In& in, long long, int, int, float (&y)[8], F32x2&) const {
    float b[8];
    in.a.get(y);
    in.b.get(b);
#pragma unroll
    for (int j = 0; j < 8; j += 2) f2_split(f2_mul(activation2<kAct>(f2(y[j], y[j + 1])), f2(b[j], b[j + 1])), y[j], y[j + 1]);
  }
  __device__ __forceinline__ float factor(float) const { return 1.f; }
};

// ---- the same for rows of whole groups of 16 bf16 elements that start on 32 bytes: load() and get() of the group at element `at`, column `c`.  The rows of all
// inputs (and of h) have one stride.
struct Raw16 {
  uint32_t u[8];
  // (Volatile: not ahead of chain_wait().)  What is read once stays out of the L1: a norm with residual of 16384 x 4096 then takes 73 us, not 83.  kAgain: every row reads it (a norm's weight).
  template <bool kAgain = false>
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (kAgain)
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
          : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
          : "l"(p));
    else
      asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
          : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
          : "l"(p));
  }
  __device__ __forceinline__ void store(void* p) const {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]),
                 "r"(u[7]), "l"(p)
                 : "memory");
  }
  __device__ __forceinline__ F32x2 pair(int j) const { return f2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xFFFF0000u)); }
};
constexpr int kMostParts = 5;
struct Plain16 {  // rows of up to five matrices, one behind the other: those from row end[i - 1] on lie `off[i]` elements from where x would have them
  const __nv_bfloat16* x;
  int end[kMostParts - 1];
  long long off[kMostParts];
  struct In {
    Raw16 x;
  };
  static constexpr bool kSum = false, kTwoBlocks = false;
  __device__ __forceinline__ void load(In& in, long long at, int row) const {
    long long o = off[0];
#pragma unroll
    for (int i = 0; i < kMostParts - 1; ++i)
      if (row >= end[i]) o = off[i + 1];
    in.x.load(x + at + o);
  }
  __device__ __forceinline__ void get(const In& in, long long, int, float (&y)[16], F32x2&) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f2_split(in.x.pair(j), y[2 * j], y[2 * j + 1]);
  }
  __device__ __forceinline__ float factor(float) const { return 1.f; }
};
template <bool kResidual, bool kW32>
struct Norm16 {
  const __nv_bfloat16 *x, *r;
  __nv_bfloat16* h;
  const void* w;
  float w_offset, eps, per_col;
  struct In {
    Raw16 x, r;
  };
  static constexpr bool kSum = true, kTwoBlocks = true;
  __device__ __forceinline__ void load(In& in, long long at, int) const {
    in.x.load(x + at);
    if constexpr (kResidual) in.r.load(r + at);
  }
  __device__ __forceinline__ void get(const In& in, long long at, int c, float (&y)[16], F32x2& ss) const {
    Raw16 sum = in.x;
    if constexpr (kResidual) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // the sum in the rows' type is what goes on, here too
        float a, b;
        f2_split(f2_add(in.x.pair(j), in.r.pair(j)), a, b);
        sum.u[j] = pack_bf16x2(a, b);
      }
      sum.store(h + at);
    }
    Raw16 w0, w1;
    if (w != nullptr) {  // from the L1, row after row; from the L2 beside a residual, where the L1 is worth less than its traffic (83 us instead of 73)
      w0.template load<!kResidual>(kW32 ? static_cast<const void*>(static_cast<const float*>(w) + c) : static_cast<const void*>(static_cast<const __nv_bfloat16*>(w) + c));
      if constexpr (kW32) w1.template load<!kResidual>(static_cast<const float*>(w) + c + 8);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      F32x2 v = sum.pair(j);
      ss = f2_fma(v, v, ss);
      if (w != nullptr) {
        F32x2 f;
        if constexpr (kW32) f = f2(__uint_as_float(j < 4 ? w0.u[2 * j % 8] : w1.u[2 * j % 8]), __uint_as_float(j < 4 ? w0.u[(2 * j + 1) % 8] : w1.u[(2 * j + 1) % 8]));
        else f = w0.pair(j);
        if (w_offset != 0.f) f = f2_add(f, f2(w_offset, w_offset));
        v = f2_mul(v, f);
      }
      f2_split(v, y[2 * j], y[2 * j + 1]);
    }
  }
  __device__ __forceinline__ float mean(float ss) const { return ss * per_col + eps; }
  __device__ __forceinline__ float factor(float ss) const { return rsqrtf(mean(ss)); }
  __device__ __forceinline__ Normed<__nv_bfloat16> normed(long long ld) const { return {kResidual ? h : x, w, ld, kW32, w_offset, eps}; }
};
template <int kAct>
struct Glu16 {
  const __nv_bfloat16 *g, *u;
  struct In {
    Raw16 g, u;
  };
  static constexpr bool kSum = false, kTwoBlocks = true;
  __device__ __forceinline__ void load(In& in, long long at, int) const {
    in.g.load(g + at);
    in.u.load(u + at);
  }
  __device__ __forceinline__ void get(const In& in, long long, int, float (&y)[16], F32x2&) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f2_split(f2_mul(activation2<kAct>(in.g.pair(j)), in.u.pair(j)), y[2 * j], y[2 * j + 1]);
  }
  __device__ __forceinline__ float factor(float) const { return 1.f; }
};

// The largest of three magnitudes, NaN if one of them is
__device__ __forceinline__ float largest_of(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Eight whole numbers as bytes.  Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves it in the low bits.
__device__ __forceinline__ uint2 whole8(const float* y, float top, float inv) {
  constexpr float kMagic = 12582912.f;
  uint32_t b[8];
  float far = 0.f;  // how far the furthest lies from its whole number
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const F32x2 v = f2(y[j], y[j + 1]), k = f2(inv, inv);
    const F32x2 m = f2_fma(v, k, f2(kMagic, kMagic));
    const F32x2 q = f2_fma(m, f2(-1.f, -1.f), f2(kMagic, kMagic));
    float d0, d1, m0, m1;
    f2_split(f2_fma(v, k, q), d0, d1);
    f2_split(m, m0, m1);
    far = largest_of(far, d0, d1);
    b[j] = __float_as_uint(m0);
    b[j + 1] = __float_as_uint(m1);
  }
  if (far > 0.4999f) {  // is 127 y above, on or below the border of two whole numbers, (floor + 1/2) max |y|?
    const bool large = top >= 1e30f;  // both sides 2^-20 times, so that neither runs over
    const float t = large ? top * 9.5367431640625e-07f : top, by = large ? 127.f * 9.5367431640625e-07f : 127.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float border = floorf(y[j] * inv) + 0.5f;
      const float above = fmaf(-border, t, y[j] * by);
      b[j] = __float_as_uint(__fadd_rn(above > 0.f ? border + 0.5f : above < 0.f ? border - 0.5f : border, kMagic));
    }
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return o;
}

constexpr int kRowWarps = 4;  // of a block whose warps have a row each

constexpr int kHeldGroups = 2;   // groups of eight per thread of a block that has a row
constexpr int kMostThreads = 1024;

// What the threads of a row agree on: its largest magnitude (as bits, which order infinities and NaN last) and its factor.
struct RowScale {
  float most, inv, scale;
  bool live;
  __device__ __forceinline__ RowScale(uint32_t top, float f) {
    most = __uint_as_float(top);
    const bool finite = top < 0x7F800000u && f == f;
    live = finite && most * f >= kTiny && most >= kLeast;
    // (the quick quotient is good for divisors up to 2^126; 1e30 keeps the quotient a normal number, too)
    inv = !live ? 0.f : most < 1e30f ? __fdividef(127.f, most) : 127.f / most;
    scale = most * f;
    if (!live) scale = finite ? 0.f : __uint_as_float(0x7FC00000u);
  }
  __device__ __forceinline__ float step() const {  // (NaN stays)
    const float s = scale / 127.f;
    return s > kMostScale ? kMostScale : s;
  }
  __device__ __forceinline__ void put(int8_t* out, const float (&v)[8]) const {
    *reinterpret_cast<uint2*>(out) = live ? whole8(v, most, inv) : make_uint2(0, 0);
  }
};
__device__ __forceinline__ void note(float& largest, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) largest = largest_of(largest, v[j], v[j + 1]);
}
// The maximum and sum over a block, through `tops` and `sums` [32], in which the numbers of warps that do not exist are 0.
template <bool kSum>
__device__ __forceinline__ void reduce_block(uint32_t& top, float& ss, uint32_t* tops, float* sums) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    tops[warp] = top;
    if constexpr (kSum) sums[warp] = ss;
  }
  __syncthreads();
  top = 0;
  ss = 0.f;
  for (int i = 0; i < warps; i += 4) {
    const uint4 v = reinterpret_cast<const uint4*>(tops)[i / 4];
    top = max(max(top, max(v.x, v.y)), max(v.z, v.w));
    if constexpr (kSum) {
      const float4 a = reinterpret_cast<const float4*>(sums)[i / 4];
      ss += (a.x + a.y) + (a.z + a.w);
    }
  }
}
template <bool kSum>
__device__ __forceinline__ float warp_ss(F32x2 ss2) {
  if constexpr (!kSum) return 0.f;
  float a, b;
  f2_split(ss2, a, b);
  return warp_sum(a + b);
}

// Rows whose sum of squares left the range of fp32: elements from some 1e19 on and, with an eps below 2^-90, those that are smaller than that.  (`top`: of a row
// without NaN and not of zeros; it may have run over itself.)  One thread of a row notes them by a scale that no row has, and when a block is through with its
// rows it makes them again, so that the loop over the rows holds no code of this.
constexpr float kNoted = -1.f;
template <class Src>
__device__ __forceinline__ float noted(const Src& src, const RowScale& r, uint32_t top, float ss, int* again) {
  if constexpr (Src::kSum) {
    if (!(src.mean(ss) >= 0x1p-90f && src.mean(ss) <= 3.402823466e+38f) && top != 0 && top <= 0x7F800000u) {
      *again = 1;
      return kNoted;
    }
  }
  return r.step();
}
// All threads of a block come here with the rows that their block or (kWarp) warp had.
template <bool kWarp, typename T>
__device__ __forceinline__ void rows_in_64_bits(Normed<T> src, long long row, long long step, long long rows, int cols, int8_t* q, long long ldq, float* scale) {
  __shared__ double s_most[32], s_sums[32];
  const int lane = threadIdx.x & 31, t = kWarp ? lane : static_cast<int>(threadIdx.x), group = kWarp ? 32 : static_cast<int>(blockDim.x);
#pragma unroll 1
  for (; row < rows; row += step) {
    if (scale[row] != kNoted) continue;
    double most = 0.0, sum = 0.0;
#pragma unroll 1
    for (int c = t; c < cols; c += group) {
      const double e = src.element(row, c), y = fabs(e * src.weight(c));
      most = y > most ? y : most;
      sum += e * e;
    }
#pragma unroll 1
    for (int i = 16; i > 0; i /= 2) {
      const double other = __shfl_xor_sync(0xffffffffu, most, i);
      most = other > most ? other : most;
      sum += __shfl_xor_sync(0xffffffffu, sum, i);
    }
    if constexpr (!kWarp) {
      if (lane == 0) {
        s_most[threadIdx.x >> 5] = most;
        s_sums[threadIdx.x >> 5] = sum;
      }
      __syncthreads();
      sum = 0.0;
#pragma unroll 1
      for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
        most = s_most[i] > most ? s_most[i] : most;
        sum += s_sums[i];
      }
    }
    const double top = most / sqrt(sum / cols + static_cast<double>(src.eps));  // of the normed row
    const bool finite = most <= 1.7e308 && sum <= 1.7e308 && top == top, live = finite && top >= kTiny;
#pragma unroll 1
    for (int c = t; c < cols; c += group)
      q[row * ldq + c] = live ? static_cast<int8_t>(__double2int_rn(127.0 * (static_cast<double>(src.element(row, c)) * src.weight(c)) / most)) : 0;
    if constexpr (!kWarp) __syncthreads();  // the partial results are read, and so is the note
    else __syncwarp();
    if (t == 0) {
      const double s = top / 127.0;
      scale[row] = live ? static_cast<float>(s > kMostScale ? kMostScale : s) : finite ? 0.f : __uint_as_float(0x7FC00000u);
    }
  }
}

// The same as a function of its own, where the loop over the rows is short of registers: norms with residual of 8192 x 11007 take 312 us, 376 with it in line (317 without
// it); those without a residual 185 and 178 (180).
template <bool kWarp, typename T>
__device__ __noinline__ void rows_in_64_bits_apart(Normed<T> src, long long row, long long step, long long rows, int cols, int8_t* q, long long ldq, float* scale) {
  rows_in_64_bits<kWarp>(src, row, step, rows, cols, q, ldq, scale);
}

// Few rows, and rows that lie anywhere.  kWarp: a row per warp, else a row per block.  kChunks: groups of eight elements per thread, held in registers; 0:
// any number of them, each made twice.  A block goes through rows far apart and starts the reads of its next row before it reduces and writes the one it
// has.  q has room for whole groups of eight up to the end of its row stride.
template <class Src, bool kWarp, int kChunks, int kThreads>
__global__ void __launch_bounds__(kThreads) quantize_kernel(Src src, long long rows, int cols, int8_t* __restrict__ q, long long ldq,
                                                                                        float* __restrict__ scale) {
  __shared__ __align__(16) uint32_t s_top[2][32];
  __shared__ __align__(16) float s_ss[2][32];
  __shared__ int s_again;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = kWarp ? lane : static_cast<int>(threadIdx.x);
  const int group = kWarp ? 32 : static_cast<int>(blockDim.x);
  const long long step = kWarp ? static_cast<long long>(gridDim.x) * kRowWarps : gridDim.x;
  long long row = kWarp ? static_cast<long long>(blockIdx.x) * kRowWarps + warp : blockIdx.x;
  if constexpr (!kWarp) {
    if (threadIdx.x < 32) {
      s_top[0][lane] = s_top[1][lane] = 0;
      s_ss[0][lane] = s_ss[1][lane] = 0.f;
    }
  }
  if constexpr (Src::kSum) {
    if (threadIdx.x == 0) s_again = 0;
  }
  if constexpr (Src::kSum || !kWarp) __syncthreads();
  chain_wait();
  constexpr int kHeld = kChunks > 0 ? kChunks : 1;
  const int limit = (cols + 255) / 256 * 256;  // whole warps take part to the end of a row
  typename Src::In in[kHeld];
  auto load = [&](long long at) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (t + i * group) * 8;
      src.load(in[i], at, c, cols - c);
    }
  };
  if (row < rows) load(row);
  for (int odd = 0; row < rows; row += step, odd ^= 1) {
    float y[kHeld][8];
    F32x2 ss2 = f2(0.f, 0.f);
    float largest = 0.f;
    if constexpr (kChunks > 0) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = (t + i * group) * 8;
        src.get(in[i], row, c, cols - c, y[i], ss2);
        note(largest, y[i]);
      }
      if (row + step < rows) load(row + step);
    } else {
      for (int c = t * 8; c < limit; c += group * 8) {
        src.load(in[0], row, c, cols - c);
        src.get(in[0], row, c, cols - c, y[0], ss2);
        note(largest, y[0]);
      }
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
    float ss = warp_ss<Src::kSum>(ss2);
    // (one barrier per row: what this row reads is written again two rows on, behind the next row's)
    if constexpr (!kWarp) reduce_block<Src::kSum>(top, ss, s_top[odd], s_ss[odd]);
    const RowScale r(top, src.factor(ss));
    int8_t* out = q + row * ldq;
    if constexpr (kChunks > 0) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = (t + i * group) * 8;
        if (c < cols) r.put(out + c, y[i]);
      }
    } else {
      for (int c = t * 8; c < limit; c += group * 8) {
        F32x2 again = f2(0.f, 0.f);
        src.load(in[0], row, c, cols - c);
        src.get(in[0], row, c, cols - c, y[0], again);
        if (c < cols) r.put(out + c, y[0]);
      }
    }
    if (t == 0) scale[row] = noted(src, r, top, ss, &s_again);
  }
  if constexpr (Src::kSum) {
    __syncthreads();  // what the block has written can be read
    row = kWarp ? static_cast<long long>(blockIdx.x) * kRowWarps + warp : blockIdx.x;
    if (s_again != 0) {
      if constexpr (Src::kWide) rows_in_64_bits_apart<kWarp>(src.normed(0), row, step, rows, cols, q, ldq, scale);
      else rows_in_64_bits<kWarp>(src.normed(0), row, step, rows, cols, q, ldq, scale);
    }
  }
}

// Aligned rows of whole groups of 16 elements, a thread has one: 32 bytes of each input in one load.  kAhead: the next row's are started ahead of this one's
// reduction; else two blocks per SM of up to 768 threads.
template <class Src, bool kAhead>
__global__ void __launch_bounds__(kAhead ? kMostThreads : 768, kAhead ? 1 : 2) rows16_kernel(Src src, long long ld, int rows, int cols, int8_t* __restrict__ q, long long ldq,
                                                              float* __restrict__ scale) {
  __shared__ uint32_t s_top[2][32];
  __shared__ float s_ss[2][32];
  __shared__ int s_again;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = threadIdx.x * 16;
  const bool mine = c < cols;
  if (threadIdx.x < 32) {  // the partial results of warps that do not exist
    s_top[0][lane] = s_top[1][lane] = 0;
    s_ss[0][lane] = s_ss[1][lane] = 0.f;
    s_again = 0;
  }
  __syncthreads();
  chain_wait();
  const int step = gridDim.x;
  int row = blockIdx.x;
  long long at = row * ld + c;
  typename Src::In in;
  if (kAhead && mine) src.load(in, at, row);
  for (int odd = 0; row < rows; row += step, odd ^= 1) {
    float y[16] = {};
    F32x2 ss2 = f2(0.f, 0.f);
    float largest = 0.f;
    if (mine) {
      if constexpr (!kAhead) src.load(in, at, row);
      src.get(in, at, c, y, ss2);
#pragma unroll
      for (int j = 0; j < 16; j += 2) largest = largest_of(largest, y[j], y[j + 1]);
      at += step * ld;
      if (kAhead && row + step < rows) src.load(in, at, row + step);
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
    float ss = warp_ss<Src::kSum>(ss2);
    if (lane == 0) {
      s_top[odd][warp] = top;
      if constexpr (Src::kSum) s_ss[odd][warp] = ss;
    }
    __syncthreads();  // (one per row: what this row reads is written again two rows on, behind the next row's)
    top = __reduce_max_sync(0xffffffffu, s_top[odd][lane]);
    if constexpr (Src::kSum) ss = warp_sum(s_ss[odd][lane]);
    const RowScale r(top, src.factor(ss));
    if (mine) {
      uint2 a = make_uint2(0, 0), b = a;
      if (r.live) {
        a = whole8(y, r.most, r.inv);
        b = whole8(y + 8, r.most, r.inv);
      }
      *reinterpret_cast<uint4*>(q + row * ldq + c) = make_uint4(a.x, a.y, b.x, b.y);
    }
    if (threadIdx.x == 0) scale[row] = noted(src, r, top, ss, &s_again);
  }
  if constexpr (Src::kSum) {
    __syncthreads();  // what the block has written can be read
    if (s_again != 0) rows_in_64_bits<false>(src.normed(ld), blockIdx.x, step, rows, cols, q, ldq, scale);
  }
}

template <auto kKernel>
int resident_blocks(int threads, int shared) {  // per SM
  static int regs = 0;
  if (regs == 0) {
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, kKernel) != cudaSuccess) return 1;
    regs = (attr.numRegs + 7) / 8 * 8;
  }
  int n = 65536 / (regs * threads);
  if (n > 2048 / threads) n = 2048 / threads;
  if (n > 228 * 1024 / (shared + 2048)) n = 228 * 1024 / (shared + 2048);
  return n < 1 ? 1 : n > 32 ? 32 : n;
}

template <class Src, bool kWarp, int kChunks, int kThreads>
int launch(const Src& src, long long rows, int cols, int threads, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
  const long long blocks = kWarp ? (rows + kRowWarps - 1) / kRowWarps : rows;
  const long long most = static_cast<long long>(num_sms()) * resident_blocks<quantize_kernel<Src, kWarp, kChunks, kThreads>>(threads, 0);
  return launch_chained(quantize_kernel<Src, kWarp, kChunks, kThreads>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(threads), 0, s, src, rows, cols, q,
                        ldq, scale) == cudaSuccess
             ? kErrOk
             : kErrCuda;
}

template <class Src, bool kAhead>
int launch16(const Src& src, long long ld, long long rows, int cols, int threads, void* q, long long ldq, float* scale, void* stream) {
  const long long most = static_cast<long long>(num_sms()) * resident_blocks<rows16_kernel<Src, kAhead>>(threads, 0);
  return launch_chained(rows16_kernel<Src, kAhead>, dim3(static_cast<unsigned>(rows < most ? rows : most)), dim3(threads), 0, reinterpret_cast<cudaStream_t>(stream), src,
                        ld, static_cast<int>(rows), cols, reinterpret_cast<int8_t*>(q), ldq, scale) == cudaSuccess
             ? kErrOk
             : kErrCuda;
}

template <class Src>
int quantize16(const Src& src, long long ld, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  if (rows <= 0 || q == nullptr || scale == nullptr || (ldq & 15) || ldq < cols || (reinterpret_cast<uintptr_t>(q) & 15)) return kErrBadArg;
  const int threads = (cols / 16 + 31) / 32 * 32;
  // Of 513 to 768 threads with 64 registers an SM has one block, which stands still at its barrier; with 40, which the next row does not fit into, two.  us, one / two
  // blocks, 8192 rows of 11008: gated activation 88 / 84, norm with residual 112 / 107, without 76 / 73, but a row as it is 60 / 67.
  if constexpr (Src::kTwoBlocks) {
    if (threads > kMostThreads / 2 && threads <= 768) return launch16<Src, false>(src, ld, rows, cols, threads, q, ldq, scale, stream);
  }
  return launch16<Src, true>(src, ld, rows, cols, threads, q, ldq, scale, stream);
}

// Whether rows are of whole groups of 16 elements, few enough for a block and more than a warp takes, start on 32 bytes and have one stride.
inline bool rows16(long long rows, int cols, long long ld, std::initializer_list<std::pair<const void*, long long>> inputs) {
  if (cols % 16 != 0 || cols > 16 * kMostThreads || cols <= 512 || rows > 0x3FFFFFFF || (ld & 15)) return false;
  for (const auto& i : inputs)
    if (i.first != nullptr && ((reinterpret_cast<uintptr_t>(i.first) & 31) || i.second != ld)) return false;
  return true;
}

template <class Src>
int quantize(const Src& src, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  if (rows <= 0 || cols <= 0 || q == nullptr || scale == nullptr || (ldq & 7) || ldq < cols || (reinterpret_cast<uintptr_t>(q) & 7)) return kErrBadArg;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int8_t* o = reinterpret_cast<int8_t*>(q);
  if (cols <= 512) return launch<Src, true, 2, 32 * kRowWarps>(src, rows, cols, 32 * kRowWarps, o, ldq, scale, s);
  const int threads = ((cols + 7) / 8 + 32 * kHeldGroups - 1) / (32 * kHeldGroups) * 32;
  // The fewer threads a form is made for, the more registers each has.  us, 8192 rows: norms with residual, columns 4095 / 11007 / 14335 as forms of 1024 threads
  // 127 / 474 / 514, of 512 101, of 768 284, read twice by 512 threads (by 1024) 306 (417) for 11007 and 399 (445) for 14335; fp32, 11008 / 14336: 456 / 544, of 768 450,
  // read twice 268 (371) / 367 (424).  Gated activations of 4096 rows in fp32, 4096 / 11008 columns 38 / 136, of 512 and 768 26 / 106; in bf16, 8192 rows of 8191
  // / 11007 115 / 201, of 512 171, of 768 187.  Norms without a residual, 11007 columns 165, of 768 146.
  constexpr int kMost = Src::kMostHeld, kHalf = kMostThreads / 2;
  if (threads > kMost) {
    constexpr int kTwice = kMost < kMostThreads ? kHalf : kMostThreads;
    return launch<Src, false, 0, kTwice>(src, rows, cols, kTwice, o, ldq, scale, s);
  }
  if constexpr (Src::kWide) {
    if (threads <= kHalf) return launch<Src, false, kHeldGroups, kHalf>(src, rows, cols, threads, o, ldq, scale, s);
  }
  if constexpr (kMost >= 768) {
    if (threads <= 768 && (Src::kWide || threads > kHalf)) return launch<Src, false, kHeldGroups, 768>(src, rows, cols, threads, o, ldq, scale, s);
  }
  if constexpr (kMost == kMostThreads) return launch<Src, false, kHeldGroups, kMostThreads>(src, rows, cols, threads, o, ldq, scale, s);
  return kErrBadArg;  // (not reached: the forms above hold every row up to kMost threads)
}

// out = q * scale, rounded once, for dense rows `out`.  kGroup elements per thread: 16 of aligned rows of whole groups of 16, else 8, and those may lie
// across the ends of rows.
template <typename T, int kGroup>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ scale, long long rows,
                                                         int cols, T* __restrict__ out) {
  chain_wait();
  const long long total = rows * cols;
  const unsigned units = cols / kGroup;
  const bool narrow = total < (1ll << 32);  // a division of 32 bits is three times as fast
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i * kGroup >= total) return;
  if constexpr (kGroup == 16) {
    const long long row = narrow ? static_cast<unsigned>(i) / units : i / units;
    uint4 w;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
        : "l"(q + row * ldq + (i - row * units) * 16));
    const float s = __ldg(scale + row);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    Raw16 o[sizeof(T) / 2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t p = u[j / 2] >> (16 * (j & 1));
      const float a = static_cast<float>(static_cast<int8_t>(p)) * s, b = static_cast<float>(static_cast<int8_t>(p >> 8)) * s;
      if constexpr (sizeof(T) == 2) {
        o[0].u[j] = pack_bf16x2(a, b);
      } else {
        o[j / 4 % (sizeof(T) / 2)].u[2 * j % 8] = __float_as_uint(a);
        o[j / 4 % (sizeof(T) / 2)].u[(2 * j + 1) % 8] = __float_as_uint(b);
      }
    }
#pragma unroll
    for (int k = 0; k < sizeof(T) / 2; ++k) o[k].store(out + i * 16 + k * 8);
  } else {
    float v[8] = {};
    Raw<T> group;  // (groups of eight of a dense `out` start on 16 bytes)
    long long row = narrow ? static_cast<unsigned>(i * 8) / static_cast<unsigned>(cols) : i * 8 / cols;
    int c = static_cast<int>(i * 8 - row * cols);
    float s = __ldg(scale + row);
    if (c >= 4 && c + 12 <= cols) {  // three words of the row have the eight bytes; 16384 x 4095: 75 us byte by byte, 45 so
      const uintptr_t at = reinterpret_cast<uintptr_t>(q + row * ldq + c);
      const uint32_t* base = reinterpret_cast<const uint32_t*>(at & ~uintptr_t{3});
      const uint32_t shift = static_cast<uint32_t>(at & 3) * 8;
      const uint32_t w[3] = {__ldg(base), __ldg(base + 1), __ldg(base + 2)};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int8_t>(__funnelshift_r(w[j / 4], w[j / 4 + 1], shift) >> (j % 4 * 8))) * s;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (i * 8 + j < total) {
          v[j] = static_cast<float>(__ldg(q + row * ldq + c)) * s;
          if (++c == cols && i * 8 + j + 1 < total) {
            c = 0;
            s = __ldg(scale + ++row);
          }
        }
      }
    }
    group.set(v);
    const long long left = total - i * 8;
    if (left >= 8) group.store(out + i * 8, 8);
    else group.put(out + i * 8, 0, static_cast<int>(left));
  }
}

template <typename T>
int dequantize(const void* q, long long ldq, const float* scale, long long rows, int cols, void* out, cudaStream_t s) {
  const bool whole = cols % 16 == 0 && (ldq & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  const long long units = whole ? rows * (cols / 16) : (rows * cols + 7) / 8;
  if ((units + 255) / 256 > 0x7FFFFFFF) return kErrBadArg;
  const dim3 grid(static_cast<unsigned>((units + 255) / 256));  // (8 blocks per SM that go on from group to group: 36.6 us for 16384 x 4096, not 32.1)
  const int8_t* p = reinterpret_cast<const int8_t*>(q);
  const cudaError_t e = whole ? launch_chained(dequantize_kernel<T, 16>, grid, dim3(256), 0, s, p, ldq, scale, rows, cols, reinterpret_cast<T*>(out))
                              : launch_chained(dequantize_kernel<T, 8>, grid, dim3(256), 0, s, p, ldq, scale, rows, cols, reinterpret_cast<T*>(out));
  return e == cudaSuccess ? kErrOk : kErrCuda;
}

}  // namespace int8_rows
}  // namespace lvb

// Each of these writes q [rows, cols] (int8, row stride ldq: a multiple of 8 that is at least cols; the bytes from cols up to the next multiple of 8 are
// written too) and scale [rows] (fp32).  Row strides are in elements.
//
// x [rows, cols], bf16 or fp32.
extern "C" int lvb_int8_quantize(const void* x, int f32, long long ldx, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  if (x == nullptr) return kErrBadArg;
  if (f32) return quantize(Plain<float>{{x, ldx, rows, cols}}, rows, cols, q, ldq, scale, stream);
  if (rows16(rows, cols, ldx, {{x, ldx}})) {
    Plain16 src{static_cast<const __nv_bfloat16*>(x), {}, {}};
    for (int i = 0; i < kMostParts - 1; ++i) src.end[i] = 0x7FFFFFFF;
    return quantize16(src, ldx, rows, cols, q, ldq, scale, stream);
  }
  return quantize(Plain<__nv_bfloat16>{{x, ldx, rows, cols}}, rows, cols, q, ldq, scale, stream);
}

// The rows of up to five dense bf16 matrices with the same columns (a multiple of 16 from 528 to 16384; 32-byte aligned), one matrix behind the other:
// xi [ni, cols], those past the last null with no rows.
extern "C" int lvb_int8_quantize_parts(const void* x0, const void* x1, const void* x2, const void* x3, const void* x4, int n0, int n1, int n2, int n3, int n4,
                                       int cols, void* q, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  const void* x[kMostParts] = {x0, x1, x2, x3, x4};
  const int n[kMostParts] = {n0, n1, n2, n3, n4};
  Plain16 src{static_cast<const __nv_bfloat16*>(x0), {}, {}};
  long long rows = 0;
  for (int i = 0; i < kMostParts; ++i) {
    if (n[i] < 0 || (n[i] > 0 && x[i] == nullptr)) return kErrBadArg;
    src.off[i] = n[i] > 0 ? (reinterpret_cast<intptr_t>(x[i]) - reinterpret_cast<intptr_t>(x0)) / 2 - rows * cols : 0;
    rows += n[i];
    if (rows > 0x3FFFFFFF) return kErrTooLarge;
    if (i < kMostParts - 1) src.end[i] = static_cast<int>(rows);
  }
  if (n0 <= 0 || !rows16(rows, cols, cols, {{x0, cols}, {x1, cols}, {x2, cols}, {x3, cols}, {x4, cols}})) return kErrBadArg;
  return quantize16(src, cols, rows, cols, q, cols, scale, stream);
}

// The RMS norm of x (+ residual): weight [cols] (w_f32: fp32, else bf16; may be null) plus w_offset.  With a residual h = x + residual is written, in
// the type of x, and is what is normed.
extern "C" int lvb_int8_rms_norm(const void* x, const void* residual, void* h, int f32, long long ldx, long long ldr, long long ldh, const void* weight,
                                 int w_f32, float w_offset, float eps, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  using bf16 = __nv_bfloat16;
  if (x == nullptr || cols <= 0 || (residual == nullptr) != (h == nullptr)) return kErrBadArg;
  const float per_col = 1.f / static_cast<float>(cols);
  auto run = [&](auto with, auto wide) {
    constexpr bool kResidual = decltype(with)::value, kWide = decltype(wide)::value;
    if (!f32 && rows16(rows, cols, ldx, {{x, ldx}, {residual, ldr}, {h, ldh}, {weight, ldx}}))
      return quantize16(Norm16<kResidual, kWide>{static_cast<const bf16*>(x), static_cast<const bf16*>(residual), static_cast<bf16*>(h), weight, w_offset, eps, per_col},
                        ldx, rows, cols, q, ldq, scale, stream);
    auto general = [&](auto type) {
      using T = decltype(type);
      Span<T> r{};
      if (kResidual) r = Span<T>(residual, ldr, rows, cols);
      return quantize(Norm<T, kResidual>{{x, ldx, rows, cols}, r, static_cast<T*>(h), weight, ldh, w_f32, w_offset, eps, per_col}, rows, cols, q, ldq, scale, stream);
    };
    return f32 ? general(float{}) : general(bf16{});
  };
  using yes = std::true_type;
  using no = std::false_type;
  if (residual != nullptr) return w_f32 ? run(yes{}, yes{}) : run(yes{}, no{});
  return w_f32 ? run(no{}, yes{}) : run(no{}, no{});
}

// act(gate) * up; act: 0 silu, 1 gelu (tanh form), 2 gelu, 3 relu, 4 g sigmoid(1.702 g).
extern "C" int lvb_int8_glu(const void* gate, const void* up, int f32, long long ldg, long long ldu, int act, long long rows, int cols, void* q,
                            long long ldq, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  using bf16 = __nv_bfloat16;
  if (gate == nullptr || up == nullptr || act < 0 || act > 4) return kErrBadArg;
  auto run = [&](auto kind) {
    constexpr int kAct = decltype(kind)::value;
    if (f32) return quantize(Glu<float, kAct>{{gate, ldg, rows, cols}, {up, ldu, rows, cols}}, rows, cols, q, ldq, scale, stream);
    if (rows16(rows, cols, ldg, {{gate, ldg}, {up, ldu}}))
      return quantize16(Glu16<kAct>{static_cast<const bf16*>(gate), static_cast<const bf16*>(up)}, ldg, rows, cols, q, ldq, scale, stream);
    return quantize(Glu<bf16, kAct>{{gate, ldg, rows, cols}, {up, ldu, rows, cols}}, rows, cols, q, ldq, scale, stream);
  };
  switch (act) {
    case kSilu: return run(std::integral_constant<int, kSilu>{});
    case kGeluTanh: return run(std::integral_constant<int, kGeluTanh>{});
    case kGelu: return run(std::integral_constant<int, kGelu>{});
    case kRelu: return run(std::integral_constant<int, kRelu>{});
    default: return run(std::integral_constant<int, kQuickGelu>{});
  }
}

// out [rows, cols] dense, bf16 or fp32 (f32).
extern "C" int lvb_int8_dequantize(const void* q, long long ldq, const float* scale, long long rows, int cols, void* out, int f32, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  if (q == nullptr || scale == nullptr || out == nullptr || rows <= 0 || cols <= 0 || ldq < cols || (reinterpret_cast<uintptr_t>(out) & 15)) return kErrBadArg;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return f32 ? dequantize<float>(q, ldq, scale, rows, cols, out, s) : dequantize<__nv_bfloat16>(q, ldq, scale, rows, cols, out, s);
}
