// Rows held in 8 bits: whole numbers q[j] = round(127 y[j] / max |y|), ties to the even one, and one fp32 scale max |y| / 127 per row, written where
// the row is made: from the RMS norm of x (+ residual), from a gated activation, or from a row as it is.  And back: q[j] * scale.
//
// The mathematics.  A norm multiplies a row by a factor f = rsqrt(mean h^2 + eps) of its own, which leaves q as it is and joins the scale, so the sum
// of squares and the largest |h w| are taken in one pass over the row and one exchange between its threads.  127 y / max |y| is the correctly
// rounded quotient wherever rounding it to a whole number could go either way: the product with the reciprocal decides the rest, and the few
// elements that it leaves within 1e-4 of a tie are divided (the product is off by at most 127 * 2^-22).  bf16 rows need this: half of the largest
// value lies on a tie, and a row often holds it.  A row below 2^-100 is stored as zeros with scale 0 (its reciprocal could overflow); a row with an
// infinity or a NaN as zeros with scale NaN, so that everything made from it is NaN.
//
// What bounds it: memory.  One pass reads the inputs and writes 1 byte per element (and h, 2 or 4).  The threads of a row keep it in registers as
// fp32 between the reduction and the write: a warp per row up to 1024 columns, up to 1024 threads per row beyond that, and above 32768
// columns the row is read twice.
#include "common.cuh"

namespace lvb {
namespace int8_rows {

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100

enum Act : int { kSilu = 0, kGeluTanh = 1, kGelu = 2, kRelu = 3, kQuickGelu = 4 };

__device__ __forceinline__ float activation(float g, int act) {
  switch (act) {
    case kSilu: return __fdividef(g, 1.f + __expf(-g));  // 2^-20 relative, far below half a step of the 8 bits
    case kGeluTanh: return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g)));
    case kGelu: return 0.5f * g * (1.f + erff(g * 0.7071067811865476f));
    case kRelu: return g != g ? g : fmaxf(g, 0.f);
    default: return __fdividef(g, 1.f + __expf(-1.702f * g));
  }
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// Eight elements from column c on (`live` of them exist, the others are zero); 16-byte loads where the address allows.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int live, float (&v)[8]) {
  if (live >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(u[j] << 16);
      v[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < live ? __bfloat162float(p[j]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* p, int live, float (&v)[8]) {
  if (live >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < live ? p[j] : 0.f;
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, int live, const float (&v)[8]) {
  if (live >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < live) p[j] = __float2bfloat16(v[j]);
  }
}
__device__ __forceinline__ void store8(float* p, int live, const float (&v)[8]) {
  if (live >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < live) p[j] = v[j];
  }
}

// ---- where a row comes from: get() gives eight of its elements and adds what the row's factor needs to `ss`
template <typename T>
struct Plain {
  const T* x;
  long long ldx;
  __device__ __forceinline__ void get(long long row, int c, int live, float (&y)[8], float&) const { load8(x + row * ldx + c, live, y); }
  __device__ __forceinline__ float factor(float, int) const { return 1.f; }
  static constexpr bool kSum = false;
};

template <typename T>
struct Norm {
  const T* x;
  const T* r;  // may be null
  T* h;        // written where there is a residual
  const void* w;
  long long ldx, ldr, ldh;
  int w_f32;
  float w_offset, eps;
  static constexpr bool kSum = true;
  __device__ __forceinline__ void get(long long row, int c, int live, float (&y)[8], float& ss) const {
    load8(x + row * ldx + c, live, y);
    if (r != nullptr) {
      float b[8];
      load8(r + row * ldr + c, live, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] += b[j];
        if constexpr (sizeof(T) == 2) y[j] = __bfloat162float(__float2bfloat16(y[j]));  // the sum in the rows' type is what goes on, here too
      }
      store8(h + row * ldh + c, live, y);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
    if (w != nullptr) {
      float f[8];
      if (w_f32) load8(reinterpret_cast<const float*>(w) + c, live, f);
      else load8(reinterpret_cast<const __nv_bfloat16*>(w) + c, live, f);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < live) y[j] *= f[j] + w_offset;
    }
  }
  __device__ __forceinline__ float factor(float ss, int cols) const { return rsqrtf(ss / static_cast<float>(cols) + eps); }
};

template <typename T>
struct Glu {
  const T* g;
  const T* u;
  long long ldg, ldu;
  int act;
  static constexpr bool kSum = false;
  __device__ __forceinline__ void get(long long row, int c, int live, float (&y)[8], float&) const {
    float b[8];
    load8(g + row * ldg + c, live, y);
    load8(u + row * ldu + c, live, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = activation(y[j], act) * b[j];
  }
  __device__ __forceinline__ float factor(float, int) const { return 1.f; }
};

// Eight whole numbers as bytes.  Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves it in the low bits.
__device__ __forceinline__ uint2 whole8(const float (&y)[8], float top, float inv) {
  constexpr float kMagic = 12582912.f;
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = y[j] * inv;
    float m = t + kMagic;
    if (fabsf(t - (m - kMagic)) > 0.4999f) m = __fdiv_rn(y[j] * 127.f, top) + kMagic;
    b[j] = __float_as_uint(m);
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return o;
}

// G threads per row, each with kChunks groups of eight elements in registers; kChunks == 0: any number of them, each made twice.  q has room for
// whole groups of eight up to the end of its row stride.
template <class Src, int G, int kChunks>
__global__ void __launch_bounds__(G < 128 ? 128 : G) quantize_kernel(Src src, long long rows, int cols, int8_t* __restrict__ q, long long ldq,
                                                                     float* __restrict__ scale) {
  constexpr int kBlock = G < 128 ? 128 : G;
  constexpr int kWarps = G / 32;
  const int lane = threadIdx.x & 31;
  const int t = threadIdx.x % G;
  const long long row = static_cast<long long>(blockIdx.x) * (kBlock / G) + threadIdx.x / G;
  chain_wait();
  if (kWarps <= 1 && row >= rows) return;  // whole warps; a larger group is a whole CTA and has its row
  float y[kChunks > 0 ? kChunks : 1][8];
  float ss = 0.f;
  uint32_t top = 0;  // magnitudes order as their bits, infinities and NaN last
  auto note = [&](const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  };
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (t + i * G) * 8;
      if (c < cols) {
        src.get(row, c, cols - c, y[i], ss);
        note(y[i]);
      }
    }
  } else {
    for (int c = t * 8; c < cols; c += G * 8) {
      src.get(row, c, cols - c, y[0], ss);
      note(y[0]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if constexpr (Src::kSum) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  if constexpr (kWarps > 1) {
    __shared__ uint32_t s_top[32];
    __shared__ float s_ss[32];
    if (lane == 0) {
      s_top[threadIdx.x >> 5] = top;
      s_ss[threadIdx.x >> 5] = ss;
    }
    __syncthreads();
    top = lane < kWarps ? s_top[lane] : 0u;
    ss = lane < kWarps ? s_ss[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if constexpr (Src::kSum) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
  }
  const float f = src.factor(ss, cols);
  const float most = __uint_as_float(top);
  const bool finite = top < 0x7F800000u && f == f;
  const bool live = finite && most * f >= kTiny;
  const float inv = live ? 127.f / most : 0.f;
  const float s = live ? most * f / 127.f : finite ? 0.f : __uint_as_float(0x7FC00000u);
  int8_t* out = q + row * ldq;
  auto put = [&](int c, const float (&v)[8]) { *reinterpret_cast<uint2*>(out + c) = live ? whole8(v, most, inv) : make_uint2(0, 0); };
  if constexpr (kChunks > 0) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (t + i * G) * 8;
      if (c < cols) put(c, y[i]);
    }
  } else {
    for (int c = t * 8; c < cols; c += G * 8) {
      float again = 0.f;
      src.get(row, c, cols - c, y[0], again);
      put(c, y[0]);
    }
  }
  if (t == 0) scale[row] = s;
}

template <class Src, int G, int kChunks>
int launch(const Src& src, long long rows, int cols, int8_t* q, long long ldq, float* scale, cudaStream_t s) {
  constexpr int kBlock = G < 128 ? 128 : G;
  const long long blocks = (rows + kBlock / G - 1) / (kBlock / G);
  if (blocks > 0x7FFFFFFFll) return kErrTooLarge;
  return launch_chained(quantize_kernel<Src, G, kChunks>, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, src, rows, cols, q, ldq, scale) == cudaSuccess
             ? kErrOk
             : kErrCuda;
}

template <class Src>
int quantize(const Src& src, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  if (rows <= 0 || cols <= 0 || q == nullptr || scale == nullptr || (ldq & 7) || ldq < cols || (reinterpret_cast<uintptr_t>(q) & 7)) return kErrBadArg;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int8_t* o = reinterpret_cast<int8_t*>(q);
  if (cols <= 256) return launch<Src, 32, 1>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 512) return launch<Src, 32, 2>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 1024) return launch<Src, 32, 4>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 2048) return launch<Src, 128, 2>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 4096) return launch<Src, 256, 2>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 8192) return launch<Src, 512, 2>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 16384) return launch<Src, 512, 4>(src, rows, cols, o, ldq, scale, s);
  if (cols <= 32768) return launch<Src, 1024, 4>(src, rows, cols, o, ldq, scale, s);
  return launch<Src, 1024, 0>(src, rows, cols, o, ldq, scale, s);
}

// out[row, j] = q[row, j] * scale[row]; 16 elements per thread where the addresses allow, rounded once
template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ scale, long long rows,
                                                         int cols, T* __restrict__ out) {
  chain_wait();
  const int units = (cols + 7) / 8;
  const long long total = rows * units;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long row = i / units;
    const int c = static_cast<int>(i - row * units) * 8, live = min(8, cols - c);
    const int8_t* p = q + row * ldq + c;
    const float s = scale[row];
    float v[8];
    if (live == 8 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = static_cast<float>(static_cast<int8_t>(w.x >> (8 * j))) * s;
        v[4 + j] = static_cast<float>(static_cast<int8_t>(w.y >> (8 * j))) * s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < live ? static_cast<float>(p[j]) * s : 0.f;
    }
    store8(out + row * cols + c, live, v);
  }
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
  if (f32) return quantize(Plain<float>{reinterpret_cast<const float*>(x), ldx}, rows, cols, q, ldq, scale, stream);
  return quantize(Plain<__nv_bfloat16>{reinterpret_cast<const __nv_bfloat16*>(x), ldx}, rows, cols, q, ldq, scale, stream);
}

// The RMS norm of x (+ residual): weight [cols] (w_f32: fp32, else bf16; may be null) plus w_offset.  With a residual h = x + residual is written, in
// the type of x, and is what is normed.
extern "C" int lvb_int8_rms_norm(const void* x, const void* residual, void* h, int f32, long long ldx, long long ldr, long long ldh, const void* weight,
                                 int w_f32, float w_offset, float eps, long long rows, int cols, void* q, long long ldq, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  if (x == nullptr || (residual == nullptr) != (h == nullptr)) return kErrBadArg;
  if (f32)
    return quantize(Norm<float>{reinterpret_cast<const float*>(x), reinterpret_cast<const float*>(residual), reinterpret_cast<float*>(h), weight, ldx, ldr, ldh,
                                w_f32, w_offset, eps},
                    rows, cols, q, ldq, scale, stream);
  return quantize(Norm<__nv_bfloat16>{reinterpret_cast<const __nv_bfloat16*>(x), reinterpret_cast<const __nv_bfloat16*>(residual),
                                      reinterpret_cast<__nv_bfloat16*>(h), weight, ldx, ldr, ldh, w_f32, w_offset, eps},
                  rows, cols, q, ldq, scale, stream);
}

// act(gate) * up; act: 0 silu, 1 gelu (tanh form), 2 gelu, 3 relu, 4 g sigmoid(1.702 g).
extern "C" int lvb_int8_glu(const void* gate, const void* up, int f32, long long ldg, long long ldu, int act, long long rows, int cols, void* q,
                            long long ldq, float* scale, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  if (gate == nullptr || up == nullptr || act < 0 || act > 4) return kErrBadArg;
  if (f32)
    return quantize(Glu<float>{reinterpret_cast<const float*>(gate), reinterpret_cast<const float*>(up), ldg, ldu, act}, rows, cols, q, ldq, scale, stream);
  return quantize(Glu<__nv_bfloat16>{reinterpret_cast<const __nv_bfloat16*>(gate), reinterpret_cast<const __nv_bfloat16*>(up), ldg, ldu, act}, rows, cols, q, ldq,
                  scale, stream);
}

// out [rows, cols] dense, bf16 or fp32 (f32).
extern "C" int lvb_int8_dequantize(const void* q, long long ldq, const float* scale, long long rows, int cols, void* out, int f32, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_rows;
  if (q == nullptr || scale == nullptr || out == nullptr || rows <= 0 || cols <= 0 || ldq < cols) return kErrBadArg;
  const long long units = rows * ((cols + 7) / 8), most = 16ll * num_sms();
  const unsigned blocks = static_cast<unsigned>((units + 255) / 256 < most ? (units + 255) / 256 : most);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = f32 ? launch_chained(dequantize_kernel<float>, blocks, 256, 0, s, reinterpret_cast<const int8_t*>(q), ldq, scale, rows, cols,
                                             reinterpret_cast<float*>(out))
                            : launch_chained(dequantize_kernel<__nv_bfloat16>, blocks, 256, 0, s, reinterpret_cast<const int8_t*>(q), ldq, scale, rows, cols,
                                             reinterpret_cast<__nv_bfloat16*>(out));
  return e == cudaSuccess ? kErrOk : kErrCuda;
}
