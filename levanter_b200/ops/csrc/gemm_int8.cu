// Products of rows held in 8 bits: C[M,N] = (A[M,K] B[N,K]^T) scale_a[M] scale_b[N] (+ bias[N]) (+ residual[M,N]) for int8 A and B.
//
// The sums are whole numbers in 32 bits and exact (K <= 131071, as 128 * 128 * K has to fit), so their order and any split of them change nothing.
// The scales are applied once, to the sum, in fp32 (a row of very large numbers in two steps, see times_scales); then bias and residual are added and the
// result is rounded once.
//
// Three kernels, for rows of activations that are few, some or many:
//   few     up to 16 rows: a stream over the weights, which the lanes read straight into the fragments of warp-level matrix instructions;
//   stream  up to a few hundred rows: weights are the 128 rows of a tcgen05 tile and the activations its columns, K is split over a cluster whose CTAs
//           exchange their partial sums through distributed shared memory;
//   pair    256 x 256 tiles on CTA pairs (tcgen05 cta_group::2, kind::i8), persistent, accumulators double-buffered in tensor memory.
// choose() says which takes what, with both sides measured.
//
// What bounds them: few and stream read every weight once, so memory from some 100 MB of weights on (28672 x 4096, one row: 20.8 us, 5.6 TB/s), and below
// that a launch and the first loads' way (4096 x 4096, one row: 5.2 us; 64 rows of 6144 x 4096: 10.4).  pair is bound by the matrix units and, in long
// runs, by the power they draw: 8192 x 11008 x 4096 in 237 us, 3.1 Pop/s; 8192 x 4096 x 14336 with residual in
// 315.  From some 2000 columns of K down the results' way to memory counts too: 2000 x 16384 x 2048 53 us, of which the sums 39.
// Every wait is bounded (common.cuh).
#include <type_traits>

#include "cta_pair.cuh"

namespace lvb {
namespace int8_gemm {
using namespace cta_pair;

constexpr int BK = 128;      // bytes of K per stage: one 128-byte swizzled line per row
constexpr int kUmmaK = 32;   // of which one matrix instruction takes 32
constexpr int kThreads = 192;  // warp 0 TMA, warp 1 MMA and tensor memory, warps 2-5 epilogue

enum Flags : int { kOutF32 = 1, kBias = 2, kBiasF32 = 4, kResidual = 8, kResidualF32 = 16 };

struct Params {
  void* C;
  const float* scale_a;
  const float* scale_b;
  const void* bias;
  const void* residual;
  int M, N, K;
  long long ldc, ldr;
  int flags;
  int* status;
  int aligned = 0;  // 32 columns of C and of the residual from a multiple of 32 on start on 32 bytes in every row
};

// Instruction descriptor for kind::i8: signed 8-bit A and B, both K-major, 32-bit whole-number accumulator.
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_ss_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float bias_at(const Params& p, int n) {
  if (!(p.flags & kBias)) return 0.f;
  return (p.flags & kBiasF32) ? __ldg(reinterpret_cast<const float*>(p.bias) + n)
                              : __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p.bias) + n));
}
// Rows of very large numbers (bf16 reaches 3e38): sum * sa may run over where sum * sa * sb does not.  2^-32 of such a scale does not, and the 2^32 at
// the end are exact, so that other rows' results are the same bits with and without them.
constexpr float kLargeScale = 0x1p+64f, kDown = 0x1p-32f, kUp = 0x1p+32f;
__device__ __forceinline__ float times_scales(int sum, float sa, float sb, float bias) {
  const float v = static_cast<float>(sum) * sa * sb + bias;
  return fabsf(v) <= 3.402823466e+38f ? v : static_cast<float>(sum) * (sa * kDown) * sb * kUp + bias;
}
// One element of the result: the sum of whole numbers, its scales, bias and residual.
__device__ __forceinline__ void finish(const Params& p, int m, int n, int sum, float sa, float sb, float bias) {
  float v = times_scales(sum, sa, sb, bias);
  if (p.flags & kResidual)
    v += (p.flags & kResidualF32) ? __ldg(reinterpret_cast<const float*>(p.residual) + m * p.ldr + n)
                                  : __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p.residual) + m * p.ldr + n));
  if (p.flags & kOutF32) reinterpret_cast<float*>(p.C)[m * p.ldc + n] = v;
  else reinterpret_cast<__nv_bfloat16*>(p.C)[m * p.ldc + n] = __float2bfloat16(v);
}
// The same for the first `live` of kRows rows from m on in one column, whose lanes' neighbours hold the neighbouring columns: 32 of them write a line of
// a row together.  `in`: the column exists.  finish_rows() takes numbers that have their scales and bias, finish_column() sums and the rows' scales in shared memory.
template <int kRows, class Value>
__device__ __forceinline__ void finish_rows(const Params& p, int m, int live, int n, bool in, Value value) {
  if (!in) return;
  float v[kRows];
  if (p.flags & kResidual) {
    // all loads ahead of the first use, and none behind a condition of its own, which would make them wait for one another: rows that do not exist read the last
    const int last = live - 1;
    if (p.flags & kResidualF32) {
      const float* r = reinterpret_cast<const float*>(p.residual) + m * p.ldr + n;
#pragma unroll
      for (int j = 0; j < kRows; ++j) v[j] = __ldg(r + min(j, last) * p.ldr);
    } else {
      const unsigned short* r = reinterpret_cast<const unsigned short*>(p.residual) + m * p.ldr + n;
      unsigned short h[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j) h[j] = __ldg(r + min(j, last) * p.ldr);
#pragma unroll
      for (int j = 0; j < kRows; ++j) v[j] = __uint_as_float(static_cast<uint32_t>(h[j]) << 16);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) v[j] += value(j);
  } else {
#pragma unroll
    for (int j = 0; j < kRows; ++j) v[j] = value(j);
  }
  auto put = [&](auto* o, auto whole) {
#pragma unroll
    for (int j = 0; j < kRows; ++j, o += p.ldc) {
      if (decltype(whole)::value || j < live) {
        if constexpr (sizeof(*o) == 4) *o = v[j];
        else *o = __float2bfloat16(v[j]);
      }
    }
  };
  if (p.flags & kOutF32) {
    float* o = reinterpret_cast<float*>(p.C) + m * p.ldc + n;
    if (live >= kRows) put(o, std::true_type{});
    else put(o, std::false_type{});
  } else {
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.C) + m * p.ldc + n;
    if (live >= kRows) put(o, std::true_type{});
    else put(o, std::false_type{});
  }
}
template <int kRows>
__device__ __forceinline__ void finish_column(const Params& p, int m, int live, int n, bool in, const int (&sum)[kRows], const float* sa, float sb, float bias) {
  finish_rows<kRows>(p, m, live, n, in, [&](int j) { return times_scales(sum[j], sa[j], sb, bias); });
}
// Brings `columns` of the residual from row m, column n on (which exist) into the L2 while the sums are still being made.
__device__ __forceinline__ void prefetch_residual(const Params& p, int m, int n, int columns) {
  const int size = (p.flags & kResidualF32) ? 4 : 2;
  const char* at = reinterpret_cast<const char*>(p.residual) + (m * p.ldr + n) * size;
  for (int i = 0; i < columns * size; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i));
}

// ================================================================ few rows
// A warp takes 16 output channels and every 8th piece of 64 bytes of K.  A lane's 16 bytes of a channel are the four registers that two instructions
// of K = 32 want from it, if K is counted in the order in which the lanes hold it; the activations' bytes are read in the same order, so nothing
// passes through shared memory.  kTiles: groups of 8 rows.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// The first `live` (1 to 16 or more) of 16 bytes, zeros for the others: what lies behind a row's end does not count.
__device__ __forceinline__ uint4 first_bytes(uint4 v, int live) {
  auto keep = [live](uint32_t w, int at) { return live >= at + 4 ? w : live <= at ? 0u : w & ((1u << (8 * (live - at))) - 1u); };
  return make_uint4(keep(v.x, 0), keep(v.y, 4), keep(v.z, 8), keep(v.w, 12));
}

constexpr int kFewWarps = 8;

template <int kTiles>
__global__ void __launch_bounds__(32 * kFewWarps) few_kernel(const int8_t* __restrict__ A, const int8_t* __restrict__ B, long long lda, long long ldb, Params p) {
  constexpr int kUnroll = 4;
  __shared__ int part[kFewWarps][8 * kTiles][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const int pieces = (p.K + 63) / 64;
  const int8_t* w0 = B + min(n0 + g, p.N - 1) * ldb + 16 * t;  // channels past the end read the last one, their sums are not stored
  const int8_t* w1 = B + min(n0 + g + 8, p.N - 1) * ldb + 16 * t;
  int c[kTiles][4] = {};
  chain_wait();
  for (int i0 = warp; i0 < pieces; i0 += kFewWarps * kUnroll) {
    uint4 wa[kUnroll], wb[kUnroll], x[kUnroll][kTiles];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = (i0 + u * kFewWarps) * 64, live = p.K - k - 16 * t;
      wa[u] = wb[u] = make_uint4(0, 0, 0, 0);
      if (live > 0) {
        wa[u] = load_stream(w0 + k);
        wb[u] = load_stream(w1 + k);
      }
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        x[u][j] = make_uint4(0, 0, 0, 0);
        if (live > 0 && j * 8 + g < p.M) x[u][j] = first_bytes(__ldg(reinterpret_cast<const uint4*>(A + (j * 8 + g) * lda + 16 * t + k)), live);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        mma_s8(c[j], wa[u].x, wb[u].x, wa[u].y, wb[u].y, x[u][j].x, x[u][j].y);
        mma_s8(c[j], wa[u].z, wb[u].z, wa[u].w, wb[u].w, x[u][j].z, x[u][j].w);
      }
  }
#pragma unroll
  for (int j = 0; j < kTiles; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][j * 8 + 2 * t + (e & 1)][g + 8 * (e >> 1)] = c[j][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * kTiles; i += 32 * kFewWarps) {
    const int m = i >> 4, n = n0 + (i & 15);
    if (m >= p.M || n >= p.N) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) sum += part[w][m][i & 15];
    finish(p, m, n, sum, __ldg(p.scale_a + m), __ldg(p.scale_b + n), bias_at(p, n));
  }
}

int launch_few(const void* A, const void* B, long long lda, long long ldb, const Params& p, cudaStream_t s) {
  const int8_t *a = reinterpret_cast<const int8_t*>(A), *b = reinterpret_cast<const int8_t*>(B);
  const dim3 grid((p.N + 15) / 16), block(32 * kFewWarps);
  const cudaError_t e = p.M <= 8 ? launch_chained(few_kernel<1>, grid, block, 0, s, a, b, lda, ldb, p) : launch_chained(few_kernel<2>, grid, block, 0, s, a, b, lda, ldb, p);
  return e == cudaSuccess ? kErrOk : kErrCuda;
}

// ================================================================ some rows
// Tile: 128 channels (TMEM lanes) x TN rows of activations (TMEM columns).  CTA r of a cluster takes the r-th share of K.  Its partial sums go to the CTA
// that finishes them, a share of the rows each, so that every CTA reads, adds and writes as much as the others.
constexpr int kMaxStages = 12;

// Rows that each of `splits` CTAs finishes of `live` ones, and how far apart (in numbers) the channels of such a share lie: four rows are written at a time, and
// an odd multiple of 16 bytes lets neighbouring channels meet in no bank.
__host__ __device__ inline int exchange_share(int live, int splits) { return ((live + splits - 1) / splits + 3) / 4 * 4; }
__host__ __device__ inline int exchange_pitch(int share) { return 4 * (share / 4 | 1); }

// A copy from this CTA's shared memory to that of CTA `to` of the cluster, completion on its barrier; both are given by their place here.
__device__ __forceinline__ void bulk_copy_to(const void* dst_here, const void* src, uint32_t bytes, uint64_t* bar_here, int to) {
  uint32_t dst, bar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(dst_here)), "r"(to));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(bar_here)), "r"(to));
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(smem_u32(src)), "r"(bytes), "r"(bar)
               : "memory");
}

template <int TN>
__global__ void __launch_bounds__(kThreads, 1)
stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, Params p, int stages, int kb_per_split, int ring_bytes) {
  constexpr int kWBytes = 128 * BK;
  constexpr int kXBytes = TN * BK;
  constexpr int kStage = kWBytes + kXBytes;
  constexpr int kCols = TN < 32 ? 32 : TN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* tfull_bar = empty_bar + kMaxStages;
  uint64_t* parts_bar = tfull_bar + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(parts_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  float* s_scale = reinterpret_cast<float*>(smem + 1024);  // the rows' scales
  uint8_t* ring = smem + 2048;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int splits;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
  const int rank = static_cast<int>(cluster_ctarank());
  const int n0 = static_cast<int>(blockIdx.x) / splits * 128;
  const int m0 = static_cast<int>(blockIdx.y) * TN;
  const int k_blocks = (p.K + BK - 1) / BK;
  const int kb0 = rank * kb_per_split;
  const int n_kb = min(k_blocks, kb0 + kb_per_split) - kb0;  // at least one (the launcher sees to it)

  const int live = min(TN, p.M - m0);
  const int share = exchange_share(live, splits), pitch = exchange_pitch(share);
  const uint32_t part_bytes = 128u * pitch * 4u;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tfull_bar, 1);
    mbar_init(parts_bar, 1);
    mbar_fence_init();
    if (splits > 1) mbar_expect_tx(parts_bar, (splits - 1) * part_bytes);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc<kCols>(tmem_holder);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for ahead of the exchange) the barriers are there
  if (warp == 0 && blockIdx.y == 0 && lane < min(stages, n_kb)) tma_prefetch_2d(&tmW, (kb0 + lane) * BK, n0);  // weights: into the L2 while the kernel before ends
  chain_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = 0; kb < n_kb; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 100, stage)) break;
        uint8_t* sw = ring + stage * kStage;
        mbar_expect_tx(&full_bar[stage], kStage);
        tma_load_2d(sw, &tmW, &full_bar[stage], (kb0 + kb) * BK, n0);
        tma_load_2d(sw + kWBytes, &tmX, &full_bar[stage], (kb0 + kb) * BK, m0);
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_i8(128, TN);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = 0; kb < n_kb; ++kb) {
        ok = mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 201, stage);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sw = smem_u32(ring + stage * kStage);
        const uint64_t wdesc = make_smem_desc(sw, 16, 1024), xdesc = make_smem_desc(sw + kWBytes, 16, 1024);
#pragma unroll
        for (int k = 0; k < BK / kUmmaK; ++k) umma_i8_ss(tmem, wdesc + k * 2, xdesc + k * 2, idesc, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit(&empty_bar[stage]);
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      if (ok) umma_commit(tfull_bar);
    }
  }
  __syncwarp();
  // ---- the epilogue's operands, while the sums are made
  const int quad = warp & 3;
  const int n = n0 + quad * 32 + lane;
  const bool in = n < p.N;
  float sb = 0.f, bias = 0.f;
  if (warp >= 2) {
    for (int i = threadIdx.x - 64; i < TN; i += 128) s_scale[i] = i < live ? __ldg(p.scale_a + m0 + i) : 0.f;
    if (in) {
      sb = __ldg(p.scale_b + n);
      bias = bias_at(p, n);
    }
    if (p.flags & kResidual)
      for (int i = threadIdx.x - 64; i < live; i += 128) prefetch_residual(p, m0 + i, n0, min(128, p.N - n0));
    named_bar_sync(1, 128);
  }
  // ---- every thread: the tile's sums are complete in this CTA
  const bool ok = mbar_wait(tfull_bar, 0, abort_flag, p.status, 300, 0);
  tc_fence_after();
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  constexpr int kLoad = TN < 32 ? 16 : 32;
  auto sums = [&](int c, int (&r)[kLoad]) {
    uint32_t u[kLoad];
    if constexpr (kLoad == 32) tmem_ld_32x32(taddr + c, u);
    else tmem_ld_32x16(taddr + c, u);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < kLoad; ++j) r[j] = static_cast<int>(u[j]);
  };
  const bool all = __all_sync(0xffffffffu, ok);
  if (splits == 1) {
    if (warp >= 2 && all)
      for (int c = 0; c < live; c += kLoad) {
        int r[kLoad];
        sums(c, r);
        finish_column<kLoad>(p, m0 + c, live - c, n, in, r, s_scale + c, sb, bias);
      }
  } else {
    // Rows [i share, (i + 1) share) of the tile are finished by CTA i.  A CTA writes its sums of every share, [channel][row], where its ring was, and sends
    // each to its CTA with one copy; it adds what it has itself to what the others send, which has a place of its own behind the ring.
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    uint8_t* sent = ring;
    uint8_t* got = ring + ring_bytes;
    if (warp >= 2) {
      if (all) {
        const int at = (quad * 32 + lane) * pitch;
        for (int c = 0; c < live; c += kLoad) {
          int r[kLoad];
          sums(c, r);
          int to = c / share, i = c - to * share;
#pragma unroll
          for (int j = 0; j < kLoad; j += 4) {
            if (c + j < live) *reinterpret_cast<int4*>(reinterpret_cast<int*>(sent + to * part_bytes) + at + i) = make_int4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            i += 4;
            if (i == share) {
              i = 0;
              ++to;
            }
          }
        }
      }
      fence_proxy_async_smem();
      named_bar_sync(1, 128);
      if (warp == 2 && lane < splits && lane != rank && all)
        bulk_copy_to(got + (rank < lane ? rank : rank - 1) * part_bytes, sent + lane * part_bytes, part_bytes, parts_bar, lane);
      const bool complete = __all_sync(0xffffffffu, mbar_wait(parts_bar, 0, abort_flag, p.status, 400, rank));
      if (all && complete) {
        const int first = rank * share, count = min(share, live - first);
        const int* own = reinterpret_cast<const int*>(sent + rank * part_bytes) + (quad * 32 + lane) * pitch;
        const int* other = reinterpret_cast<const int*>(got) + (quad * 32 + lane) * pitch;
        auto add = [&](int i, int* sum) {
          const int4 a = *reinterpret_cast<const int4*>(own + i);
          sum[0] = a.x; sum[1] = a.y; sum[2] = a.z; sum[3] = a.w;
          for (int s = 0; s < splits - 1; ++s) {
            const int4 v = *reinterpret_cast<const int4*>(other + s * 128 * pitch + i);
            sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
          }
        };
        int i = 0;
        for (; i + 4 < count; i += 8) {  // (a share is a multiple of four)
          int sum[8];
          add(i, sum);
          add(i + 4, sum + 4);
          finish_column<8>(p, m0 + first + i, count - i, n, in, sum, s_scale + first + i, sb, bias);
        }
        if (i < count) {
          int sum[4];
          add(i, sum);
          finish_column<4>(p, m0 + first + i, count - i, n, in, sum, s_scale + first + i, sb, bias);
        }
      }
    }
    cluster_sync_all();  // nobody leaves while its copies are read or written
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<kCols>(tmem);
  }
}

template <int TN>
int launch_stream(const void* A, const void* B, long long lda, long long ldb, const Params& p, int splits, int stages, cudaStream_t s) {
  constexpr int kStage = (128 + TN) * BK;
  const int k_blocks = (p.K + BK - 1) / BK;
  if (splits < 1) splits = 1;
  if (splits > 8) splits = 8;
  if (splits > k_blocks) splits = k_blocks;
  const int tiles = (p.N + 127) / 128 * ((p.M + TN - 1) / TN);
  const bool all_at_once = stages == 0;  // a ring that lets all CTAs run at once, up to three per SM: waves of them cost more than a short ring
  if (stages == 0 || stages > kMaxStages) stages = kMaxStages;
  int per, part, ring;
  while (true) {  // as many splits as the shared memory has room for
    per = (k_blocks + splits - 1) / splits;
    splits = (k_blocks + per - 1) / per;  // no empty share
    if (stages > per) stages = per;
    if (stages < 1) stages = 1;
    part = splits > 1 ? 128 * 4 * exchange_pitch(exchange_share(p.M < TN ? p.M : TN, splits)) : 0;
    const int per_sm = (tiles * splits + num_sms() - 1) / num_sms();
    // (one per SM: a long share of K gains by a deep ring, beside a short one the next kernel's first CTAs should have room)
    const int room = (!all_at_once || (per_sm <= 1 && (TN > 64 || per > 16)) ? 220 : per_sm <= 2 ? 110 : 72) * 1024;
    while (stages > (room < 220 * 1024 ? 3 : 1) && stages * kStage + (splits - 1) * part > room) --stages;
    ring = stages * kStage > splits * part ? stages * kStage : (splits * part + 1023) / 1024 * 1024;  // it also holds the sums that are sent
    if (ring + (splits - 1) * part <= 220 * 1024) break;
    --splits;  // (one split needs the ring alone)
  }
  // CTAs whose tensor memory does not fit beside that of others on their SM wait for it, and CTAs of clusters wait for one another: that could close a
  // circle.  A share of shared memory that is at least the share of tensor memory keeps out what would not fit; 34 KB keeps out the pairs of
  // the kernels with 256 x 256 tiles, which take all columns and all but 30 KB.
  constexpr int kCols = TN < 32 ? 32 : TN;
  constexpr int kLeast = kCols * 464 > 34 * 1024 ? kCols * 464 : 34 * 1024;
  int bytes = ring + (splits - 1) * part;
  if (bytes < kLeast) bytes = kLeast;
  CUtensorMap tmW, tmX;
  int rc = make_tmap_2d_u8(&tmW, B, p.N, p.K, ldb, 128);
  if (rc == kErrOk) rc = make_tmap_2d_u8(&tmX, A, p.M, p.K, lda, TN);
  if (rc != kErrOk) return rc;
  rc = allow_shared<stream_kernel<TN>>(232448);
  if (rc != kErrOk) return rc;
  const long long row_tiles = (p.M + TN - 1) / TN;
  if (row_tiles > 65535) return kErrTooLarge;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.N + 127) / 128 * splits), static_cast<unsigned>(row_tiles));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 3 * 1024 + bytes;  // alignment, barriers and scales ahead of the ring
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, stream_kernel<TN>, tmW, tmX, p, stages, per, ring) == cudaSuccess ? kErrOk : kErrCuda;
}

// ================================================================ many rows
constexpr int BN = 256, BMP = 256, BMC = 128;
constexpr int kPairStage = (BMC + BN / 2) * BK;  // per CTA
constexpr int kPairStages = 6;
constexpr int kTurn = 33;  // from row to row of 32 x 32 numbers in shared memory, which are written by rows and read by columns
constexpr int kPairSmem = 1024 + kPairStages * kPairStage + 4 * BN * 4 + 4 * 32 * kTurn * 4 + (2 * kPairStages + 4) * 8 + 16;

__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int& mb, int& nb) {
  constexpr int GM = 8;  // so many row tiles stay in the L2 while the raster sweeps N (4096 x 28672 x 4096 319 us; 4 of them 348, 2 373; other sizes within 2%)
  const int group = GM * tiles_n, g = t / group, first = g * GM, gm = min(GM, tiles_m - first), r = t - g * group;
  mb = first + r % gm;
  nb = r / gm;
}

// 32 bytes of a row at a time: whole sectors (16 bytes at a time 8192 x 11008 x 4096 takes 277 us instead of 237; by way of shared memory, so that four lanes write
// 64 bytes of a row together, 265; eight epilogue warps instead of four 291).
struct Line {
  uint32_t u[8];
  __device__ __forceinline__ void load(const void* p) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                 : "l"(p));
  }
  __device__ __forceinline__ void store(void* p) const {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]),
                 "r"(u[7]), "l"(p)
                 : "memory");
  }
};
// 32 columns of the residual in the lane's row, which are read while the 32 columns before them are written.
struct Ahead {
  Line l[4];
  __device__ __forceinline__ void load(const Params& p, int m, int n) {
    const long long at = m * p.ldr + n;
    if (p.flags & kResidualF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) l[i].load(reinterpret_cast<const float*>(p.residual) + at + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) l[i].load(reinterpret_cast<const __nv_bfloat16*>(p.residual) + at + 16 * i);
    }
  }
  __device__ __forceinline__ void add(float (&v)[32], bool f32) const {
    if (f32) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(l[j / 8].u[j % 8]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        const uint32_t w = l[j / 16].u[j % 16 / 2];
        v[j] += __uint_as_float(w << 16);
        v[j + 1] += __uint_as_float(w & 0xFFFF0000u);
      }
    }
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_scale = reinterpret_cast<float*>(smem + kPairStages * kPairStage);  // the columns' scales, of one tile and the next
  float* s_bias = s_scale + 2 * BN;
  float* s_turn = s_scale + 4 * BN;  // 32 x 32 numbers of every epilogue warp
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_turn + 4 * 32 * kTurn);
  uint64_t* empty_bar = full_bar + kPairStages;
  uint64_t* tfull_bar = empty_bar + kPairStages;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  const int tiles_m = (p.M + BMP - 1) / BMP, tiles_n = (p.N + BN - 1) / BN, tiles = tiles_m * tiles_n;
  const int k_blocks = (p.K + BK - 1) / BK;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(n_clusters_x());

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 8);  // one arrival per epilogue warp of either CTA
    }
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair<2 * BN>(tmem_holder);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anything is signalled on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  chain_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int mb, nb;
        tile_coords(t, tiles_m, tiles_n, mb, nb);
        const int m0 = mb * BMP + static_cast<int>(cta) * BMC, n0 = nb * BN + static_cast<int>(cta) * (BN / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.status, 100, stage);
          if (!ok) break;
          uint8_t* sa = smem + stage * kPairStage;
          if (cta == 0) mbar_expect_tx(&full_bar[stage], 2 * kPairStage);  // both CTAs' loads of this stage
          tma_load_2d_pair(sa, &tmA, &full_bar[stage], kb * BK, m0);
          tma_load_2d_pair(sa + BMC * BK, &tmB, &full_bar[stage], kb * BK, n0);
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && cta == 0) {
      constexpr uint32_t idesc = make_idesc_i8(BMP, BN);
      int stage = 0, buf = 0;
      uint32_t phase = 0, tphase = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        ok = mbar_wait(&tempty_bar[buf], tphase ^ 1, abort_flag, p.status, 200, buf);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, abort_flag, p.status, 201, stage);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kPairStage);
          const uint64_t adesc = make_smem_desc(sa, 16, 1024), bdesc = make_smem_desc(sa + BMC * BK, 16, 1024);
#pragma unroll
          for (int k = 0; k < BK / kUmmaK; ++k) umma_i8_ss_pair(tmem_base + buf * BN, adesc + k * 2, bdesc + k * 2, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit_pair(&empty_bar[stage]);
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair(&tfull_bar[buf]);
        if (++buf == 2) { buf = 0; tphase ^= 1; }
      }
    }
  } else {
    // epilogue: a lane has one row of this CTA's 128 and sees it 32 columns at a time
    const int quad = warp & 3;
    float* turn = s_turn + quad * (32 * kTurn);
    int buf = 0;
    uint32_t tphase = 0;
    bool alive = true;
    for (int t = first; t < tiles; t += step) {
      int mb, nb;
      tile_coords(t, tiles_m, tiles_n, mb, nb);
      const int m = mb * BMP + static_cast<int>(cta) * BMC + quad * 32 + lane;
      const bool in = m < p.M;
      float sa = in ? __ldg(p.scale_a + m) : 0.f;
      const bool large = fabsf(sa) > kLargeScale, any_large = __any_sync(0xffffffffu, large);  // as in times_scales()
      if (large) sa *= kDown;
      float* sb = s_scale + buf * BN;  // (the tile before the last one read it, and all four warps have been at a barrier since)
#pragma unroll
      for (int j = 0; j < BN; j += 128) {
        const int at = j + static_cast<int>(threadIdx.x) - 64;
        const bool there = nb * BN + at < p.N;
        sb[at] = there ? __ldg(p.scale_b + nb * BN + at) : 0.f;
        if (p.flags & kBias) s_bias[buf * BN + at] = there ? bias_at(p, nb * BN + at) : 0.f;
      }
      if (in && (p.flags & kResidual)) prefetch_residual(p, m, nb * BN, min(BN, p.N - nb * BN));
      const int m0 = m - lane, rows = min(32, p.M - m0);
      Ahead residual;
      if ((p.flags & kResidual) && p.aligned && nb * BN + 32 <= p.N) residual.load(p, min(m, p.M - 1), nb * BN);
      named_bar_sync(1, 128);
      if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&tfull_bar[buf], tphase, abort_flag, p.status, 300, buf));
      if (!alive) continue;  // the other warps wait for this one at the barrier above, tile by tile
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + buf * BN;
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        const int n0 = nb * BN + c;
        if (n0 >= p.N || rows <= 0) break;
        uint32_t r[32];
        tmem_ld_32x32(taddr + c, r);
        tmem_ld_wait();
        const int cols = min(32, p.N - n0);
        float v[32];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 f = *reinterpret_cast<const float4*>(sb + c + 4 * q);
          v[4 * q] = static_cast<float>(static_cast<int>(r[4 * q])) * sa * f.x;
          v[4 * q + 1] = static_cast<float>(static_cast<int>(r[4 * q + 1])) * sa * f.y;
          v[4 * q + 2] = static_cast<float>(static_cast<int>(r[4 * q + 2])) * sa * f.z;
          v[4 * q + 3] = static_cast<float>(static_cast<int>(r[4 * q + 3])) * sa * f.w;
        }
        if (any_large) {
          const float up = large ? kUp : 1.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= up;
        }
        if (p.flags & kBias) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 f = *reinterpret_cast<const float4*>(s_bias + buf * BN + c + 4 * q);
            v[4 * q] += f.x; v[4 * q + 1] += f.y; v[4 * q + 2] += f.z; v[4 * q + 3] += f.w;
          }
        }
        if (cols < 32 || !p.aligned) {
          // Rows that start anywhere, and the last columns: through shared memory, so that the lanes hold neighbouring columns of one row
#pragma unroll
          for (int j = 0; j < 32; ++j) turn[lane * kTurn + j] = v[j];
          __syncwarp();
          const float* column = turn + lane;
          finish_rows<32>(p, m0, rows, n0 + lane, lane < cols, [&](int i) { return column[i * kTurn]; });
          __syncwarp();
          continue;
        }
        if (p.flags & kResidual) {
          residual.add(v, p.flags & kResidualF32);
          if (n0 + 64 <= p.N && c + 32 < BN) residual.load(p, min(m, p.M - 1), n0 + 32);  // the next 32 columns
        }
        if (!in) continue;
        if (p.flags & kOutF32) {
          float* o = reinterpret_cast<float*>(p.C) + m * p.ldc + n0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            Line l;
#pragma unroll
            for (int j = 0; j < 8; ++j) l.u[j] = __float_as_uint(v[8 * i + j]);
            l.store(o + 8 * i);
          }
        } else {
          __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.C) + m * p.ldc + n0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            Line l;
#pragma unroll
            for (int j = 0; j < 8; ++j) l.u[j] = pack_bf16x2(v[16 * i + 2 * j], v[16 * i + 2 * j + 1]);
            l.store(o + 16 * i);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&tempty_bar[buf]);
      if (++buf == 2) { buf = 0; tphase ^= 1; }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves or frees tensor memory while its peer may still signal or accumulate into it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair<2 * BN>(tmem_base);
  }
}

int launch_pair(const void* A, const void* B, long long lda, long long ldb, Params p, cudaStream_t s) {
  auto whole = [](const void* x, long long ld, bool f32) { return (reinterpret_cast<uintptr_t>(x) & 31) == 0 && (ld & (f32 ? 7 : 15)) == 0; };
  p.aligned = whole(p.C, p.ldc, p.flags & kOutF32) && (!(p.flags & kResidual) || whole(p.residual, p.ldr, p.flags & kResidualF32));
  CUtensorMap tmA, tmB;
  int rc = make_tmap_2d_u8(&tmA, A, p.M, p.K, lda, BMC);
  if (rc == kErrOk) rc = make_tmap_2d_u8(&tmB, B, p.N, p.K, ldb, BN / 2);
  if (rc != kErrOk) return rc;
  rc = allow_shared<pair_kernel>(kPairSmem);
  if (rc != kErrOk) return rc;
  static int pairs = 0;  // as many as are resident at once; a GPC with an odd number of SMs has one that no pair takes
  if (pairs == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (num_sms() / 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, pair_kernel, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = num_sms() / 2;
    }
    pairs = n;
  }
  const long long tiles = static_cast<long long>((p.M + BMP - 1) / BMP) * ((p.N + BN - 1) / BN);
  if (tiles > 0x3FFFFFFF) return kErrTooLarge;
  const unsigned grid = 2u * static_cast<unsigned>(tiles < pairs ? tiles : pairs);
  return launch_chained(pair_kernel, dim3(grid), dim3(kThreads), kPairSmem, s, tmA, tmB, p) == cudaSuccess ? kErrOk : kErrCuda;
}

// Which form (us, weights out of the cache).  few / stream: 1 row, 768 x 768 2.0 / 3.2, 2304 x 768 2.6 / 3.3, 2048 x 2048 4.4 / 3.7, 4096 x 4096 7.8 / 5.3; 16 rows, 2304 x 768
// 3.3 / 3.6.  stream by tiles of 128 rows / of 256 / pair: 512 rows, 2304 x 768 5.0 / 6.6 / 9.6, 4096 x 4096 13.1 / 15.0 / 15.6; 300 rows, 8192 x 2048 (more than a wave of
// the first) 11.2 / 10.7 / 11.8; 400 rows, 14336 x 4096 34 / 36 / 27, 4096 x 14336 36 / 42 / 37; 128 rows, 28672 x 4096 24 / 36 / 30.
// Splits of K in the stream form.  A CTA gets 16 KB of weights per 0.28 us wherever they come from, so fewer than some 110 CTAs do
// not keep the memory busy, and all that run should run at once; a split costs a start, the exchange of its sums (which grows with the rows) and the rows
// of activations once more.  us for 1, 2, 4, 8 splits: 4096 x 4096, 1 row 10.8, 7.8, 5.3, 6.4, 64 rows 11.6, 10.4, 8.2, 20, 128 rows 12.3, 13.0, 10.9; 6144 x 4096, 16
// rows 11.2, 8.7, 6.9, 7.9; 8192 x 2048, 16 rows 7.4, 5.7, 6.3, 10.3; 512 x 8192, 1 row 19.5, 11.4, 7.0, 5.0; 28672 x 4096, 1 row 20.7, 25, 25, 32; 4096 x 14336, 1 row 33,
// 19, 12.7, 12.1.  Where four splits end, 1 / 2 / 3 / 4 splits: 40 tiles of K = 4096, 16 rows 11.0 / 8.7 / 7.1 / 7.4, 64 rows 12.1 / 11.4 / 9.8 / 10.3; 48 tiles 11.4 / 8.8 / 8.4 / 7.8 and
// 12.5 / 11.7 / 11.2 / 10.7 (three are 144 CTAs, one per SM, but each reads a third of K); 56 11.8 / 9.4 / 9.2 / 8.6 and 12.8 / 12.2 / 11.7 / 11.1; 68 12.6 / 10.7 / 9.7 / 9.4 and 13.3 / 13.2 / 12.3 / 12.0;
// 72, whose clusters of four do not all run at once, 12.8 / 11.0 / 10.1 / 13.4 and 13.4 / 13.5 / 12.6 / 18.4.  Of K = 2048, 16 rows, 48 tiles 7.0 / 5.5 / 6.0 / 5.5, 56 7.2 / 5.5 / 6.4 / 5.9.
struct Plan {
  int form, rows, splits;  // rows: of activations per tile of the stream form
};
inline Plan choose(int M, int N, int K) {
  const int k_blocks = (K + BK - 1) / BK, sms = num_sms(), columns = (N + 127) / 128;
  if (M <= 16 && K <= 1024 && N <= 4096) return {1, 0, 0};
  if (M <= 64) {
    int splits = 1;
    if (k_blocks >= 32 ? 13 * columns <= 6 * sms : 3 * columns <= sms) splits = 4;  // 68 and 49 tiles
    else if (2 * columns <= sms && M <= 32) splits = 2;
    if (k_blocks >= 32 && (16 * columns <= sms || (k_blocks >= 96 && M <= 32 && 4 * columns <= sms))) splits = 8;
    while (splits > 1 && k_blocks < 4 * splits) splits /= 2;
    return {2, M <= 16 ? 16 : M <= 32 ? 32 : 64, splits};
  }
  const long long narrow = static_cast<long long>(columns) * ((M + 127) / 128), wide = static_cast<long long>(columns) * ((M + 255) / 256);
  if (narrow <= sms || M <= 128) {
    int splits = 1;
    if (4 * narrow <= sms && k_blocks >= (M <= 128 ? 32 : 64)) splits = 4;
    else if (2 * narrow <= sms && k_blocks >= 64) splits = 2;
    return {2, 128, splits};
  }
  return {K <= 4096 && wide <= sms ? 2 : 3, 256, 1};
}

}  // namespace int8_gemm
}  // namespace lvb

// C[M,N] (bf16, or fp32 with flag 1; row stride ldc) = (A[M,K] B[N,K]^T) scale_a[M] scale_b[N] + bias[N] (flag 2; fp32 with flag 4, else bf16)
// + residual[M,N] (flag 8; fp32 with flag 16, else bf16; row stride ldr).  A and B: int8, 16-byte aligned, row strides multiples of 16 that are at least K.
// form: 0 lets the launcher choose; 1 few (M <= 16), 2 stream, 3 pair.  tile_rows (16, 32, 64, 128 or 256), splits (at most 8), stages: of the stream form, 0
// lets the launcher choose.
extern "C" int lvb_int8_gemm(const void* A, const void* B, const float* scale_a, const float* scale_b, void* C, int M, int N, int K, long long lda,
                             long long ldb, long long ldc, int flags, const void* bias, const void* residual, long long ldr, int form, int tile_rows,
                             int splits, int stages, int* status, void* stream) {
  using namespace lvb;
  using namespace lvb::int8_gemm;
  if (M <= 0 || N <= 0 || K <= 0 || K > 131071 || (lda & 15) || (ldb & 15) || lda < K || ldb < K || ldc < N) return kErrBadArg;
  if ((reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(B) & 15) || A == nullptr || B == nullptr || C == nullptr || scale_a == nullptr ||
      scale_b == nullptr)
    return kErrBadArg;
  if (((flags & kBias) && bias == nullptr) || ((flags & kResidual) && (residual == nullptr || ldr < N))) return kErrBadArg;
  Params p{C, scale_a, scale_b, bias, residual, M, N, K, ldc, ldr, flags, status};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Plan plan = choose(M, N, K);
  if (form != 0) plan.form = form;
  if (plan.form == 1) return M <= 16 ? launch_few(A, B, lda, ldb, p, s) : kErrBadArg;
  if (plan.form == 3) return launch_pair(A, B, lda, ldb, p, s);
  if (plan.form != 2) return kErrBadArg;
  if (form != 0) plan.rows = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  if (tile_rows != 0) plan.rows = tile_rows;
  if (splits != 0) plan.splits = splits;
  switch (plan.rows) {
    case 16: return launch_stream<16>(A, B, lda, ldb, p, plan.splits, stages, s);
    case 32: return launch_stream<32>(A, B, lda, ldb, p, plan.splits, stages, s);
    case 64: return launch_stream<64>(A, B, lda, ldb, p, plan.splits, stages, s);
    case 128: return launch_stream<128>(A, B, lda, ldb, p, plan.splits, stages, s);
    case 256: return launch_stream<256>(A, B, lda, ldb, p, plan.splits, stages, s);
    default: return kErrBadArg;
  }
}
