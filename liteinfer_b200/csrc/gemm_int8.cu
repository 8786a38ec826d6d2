// out[M, N] = x[M, K] @ W[N, K]^T (+ bias) with both operands in 8 bits: W is held as whole numbers w with a scale for each of its
// rows, x is quantised on the way with a scale for each of its rows (int8.cuh).
//
//   out[m, n] = (sum_k q[m, k] w[n, k]) * s_x[m] * s_w[n] (+ bias[n])
//
// The sum is exact (32-bit whole numbers: K up to 131,072 cannot overflow), so it may be cut and added up in any order; the two
// products are rounded in the order given and the result once more to the engine's type.
//
// Three kernels, by the number of rows of x (see li_linear_int8 for the rule).  Each of them starts while the quantisation ahead of it
// still runs (programmatic dependent launch); the first two ask for their first weights before they wait for it.
//   stream   few rows: the time is that of reading w once; per-warp rings of TMA copies, mma.sync m16n8k32
//   cluster  some rows, or few tiles: one 128 x 256 tile a cluster of up to four CTAs that share its k (tcgen05 kind::i8), their
//            sums added up through distributed shared memory
//   pair     many rows: persistent pairs of CTAs on 256 x 256 tiles (cta_group::2)
// The tensor-core kernels multiply with the operands' places changed: the first (128 or 256 rows) is w, the second x, whose rows a tile
// takes in sixteens (or thirty-twos), so that an odd number of rows of x pays for little padding.
#include "int8.cuh"
#include "tcgen05.cuh"

namespace li {

// ------------------------------------------------------------------------------------------------ rows in 8 bits
// kThreads a row, which they read once: 16 bytes a thread at a time stay in registers (kHeld of them; a longer row is read twice).
// Bound by memory: bytes of x in, one a number out.  Short rows share a block, or starting blocks is what takes the time (7,876 rows of
// 640: 12.9 us a block each, 5.5 eight a block).
constexpr int kQuantThreads = 256;

template <typename T, int kThreads, int kHeld>
__global__ void __launch_bounds__(kQuantThreads)
quantise_rows_kernel(const T* __restrict__ x, size_t row_stride, signed char* __restrict__ q, int q_stride, float* __restrict__ scale, int K,
                     int M, int vectors) {
  constexpr int N = Vec16<T>::N;
  __shared__ unsigned tops[kQuantThreads / 32];
  grid_dependency_wait();
  // Only now may the product start: it asks for its weights at once, and what the kernels ahead wrote (those weights, perhaps) is there.
  grid_launch_dependents();
  const int thread = threadIdx.x % kThreads, m = blockIdx.x * (kQuantThreads / kThreads) + threadIdx.x / kThreads;
  if (kThreads == 32 && m >= M) return;
  const T* row = x + (size_t)min(m, M - 1) * row_stride;      // (rows of several warps stay for the barrier)
  signed char* out = q + (size_t)min(m, M - 1) * q_stride;
  // `vectors` 16-byte vectors (0 where rows are not aligned), then the rest one by one.
  Vec16<T> held[kHeld];
  unsigned top = 0;
  auto largest = [&](const Vec16<T>& v) {
#pragma unroll
    for (int e = 0; e < N; ++e) top = max(top, abs_bits(v.get(e)));
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (thread + i * kThreads < vectors) held[i] = load16(row + (size_t)(thread + i * kThreads) * N);
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (thread + i * kThreads < vectors) largest(held[i]);
  for (int i = thread + kHeld * kThreads; i < vectors; i += kThreads) largest(load16(row + (size_t)i * N));
  for (int k = vectors * N + thread; k < K; k += kThreads) top = max(top, abs_bits(to_float(row[k])));
  top = warp_max_bits(top);
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (m >= M) return;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) top = max(top, tops[threadIdx.x / kThreads * (kThreads / 32) + w]);
  }
  const float s = scale_of(top);
  const bool holds = scale_holds(s), plain = scale_plain(s);
  const float inverse = plain ? __frcp_rn(s) : 0.f;
  auto write = [&](const Vec16<T>& v, int i) {
    unsigned packed[N / 4];
    float f[N];
    unpack16(v, f);
#pragma unroll
    for (int w = 0; w < N / 4; ++w) packed[w] = quantised4(f + 4 * w, s, inverse, plain);
    if constexpr (N == 8) *reinterpret_cast<uint2*>(out + (size_t)i * N) = make_uint2(packed[0], packed[1]);
    else *reinterpret_cast<unsigned*>(out + (size_t)i * N) = packed[0];
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (thread + i * kThreads < vectors) write(held[i], thread + i * kThreads);
  for (int i = thread + kHeld * kThreads; i < vectors; i += kThreads) write(load16(row + (size_t)i * N), i);
  for (int k = vectors * N + thread; k < q_stride; k += kThreads)
    out[k] = k < K ? (signed char)quantised(to_float(row[k]), s, holds) : 0;
  if (thread == 0) scale[m] = s;
}

template <typename T>
static int quantise_rows(const void* x, size_t row_stride, void* q, int q_stride, float* scale, int M, int K, cudaStream_t stream) {
  constexpr int N = Vec16<T>::N;
  const bool aligned = aligned16(x) && row_stride * sizeof(T) % 16 == 0;
  const int vectors = aligned ? K / N : 0;
  auto launch = [&](auto kernel, int threads) {
    const int rows = kQuantThreads / threads;
    return (int)launch_pdl(M, kernel, dim3((M + rows - 1) / rows), dim3(kQuantThreads), 0, stream, (const T*)x, row_stride, (signed char*)q, q_stride, scale,
                           K, M, vectors);
  };
  // Threads that hold a row between them, four vectors each or eight; more where there are few rows.
  if (vectors > 0 && vectors <= 128 && M > 8 * 148) return launch(quantise_rows_kernel<T, 32, 4>, 32);
  if (vectors > 0 && vectors <= 256 && M > 8 * 148) return launch(quantise_rows_kernel<T, 32, 8>, 32);
  if (vectors > 0 && vectors <= 512 && M > 4 * 148) return launch(quantise_rows_kernel<T, 128, 4>, 128);
  return vectors <= kQuantThreads ? launch(quantise_rows_kernel<T, 256, 1>, 256) : vectors <= 2 * kQuantThreads
                                                                                       ? launch(quantise_rows_kernel<T, 256, 2>, 256)
                                                                                       : launch(quantise_rows_kernel<T, 256, 4>, 256);
}

struct Int8GemmParams {
  const signed char* q;
  const float* q_scale;
  const float* w_scale;
  const void* bias;         // of the output's type, or null
  void* out;
  int M, N, K;              // K: bytes of a row of w
  int q_stride;             // at least K
  int* error_flag;
  int cols, col_tiles;      // rows of x a tile takes, and how many such tiles there are (cluster and pair)
  int stages;               // cluster
};

template <typename T>
__device__ __forceinline__ float scaled(int sum, float s_x, float s_w, const T* bias, int n) {
  const float v = __fmul_rn(__fmul_rn((float)sum, s_x), s_w);
  return bias != nullptr ? __fadd_rn(v, to_float(bias[n])) : v;
}

// ------------------------------------------------------------------------------------------------ stream
// A block walks over 16-row tiles of w; its warps split a tile's k, each with a ring of stages that one lane keeps full (two boxes of
// 16 rows x 128 bytes behind one mbarrier).  Both operands are read 16 bytes a lane with k permuted alike on both sides.
constexpr int kStreamK = 256;                       // bytes of k a stage
constexpr unsigned kStreamStage = 16 * kStreamK;

__device__ __forceinline__ uint4 lds128(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kCache > 0: a warp multiplies the same at most kCache stages' k in every tile and keeps its share of x in registers.
template <typename T, int NT, int kWarps, int kRing, int kCache>
__global__ void __launch_bounds__(kWarps * 32, NT < 4 ? 2 : 1)
gemm_int8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const Int8GemmParams p) {
  constexpr int kCols = NT * 8;
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  __shared__ int partial[kWarps][16][kCols + 1];
  __shared__ __align__(8) unsigned long long ring_bars[kWarps * kRing];
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int M = p.M, K = p.K;
  const int tiles = (p.N + 15) / 16, chunks = (K + kStreamK - 1) / kStreamK;
  const int per_tile = warp < chunks ? (chunks - warp + kWarps - 1) / kWarps : 0;       // stages of this warp: warp, warp + kWarps, ...
  const int my_tiles = (int)blockIdx.x < tiles ? (tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  const int items = my_tiles * per_tile;
  const unsigned ring = base + (unsigned)warp * kRing * kStreamStage;
  const unsigned bars = smem_addr(ring_bars) + (unsigned)warp * kRing * 8;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kRing; ++i) mbar_init(smem_addr(ring_bars) + 8u * i, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  auto request = [&](int n) {
    if (lane != 0 || n >= items) return;
    const int tile = blockIdx.x + (n / per_tile) * gridDim.x, k0 = (warp + (n % per_tile) * kWarps) * kStreamK;
    const unsigned slot = ring + (unsigned)(n % kRing) * kStreamStage, bar = bars + 8u * (n % kRing);
    mbar_expect_tx(bar, kStreamStage);
    tma_load_2d(slot, &map_w, bar, k0, tile * 16);
    tma_load_2d(slot + kStreamStage / 2, &map_w, bar, k0 + 128, tile * 16);
  };
  for (int n = 0; n < kRing - 1; ++n) request(n);
  grid_launch_dependents();
  grid_dependency_wait();

  const uint4 zero = make_uint4(0, 0, 0, 0);
  const signed char* xr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) xr[j] = p.q + (size_t)min(j * 8 + g, M - 1) * p.q_stride;
  auto load_x = [&](int c, int piece, int j) {
    const int k = (warp + c * kWarps) * kStreamK + (piece >> 1) * 128 + (2 * t + (piece & 1)) * 16;
    return k < K && j * 8 + g < M ? *reinterpret_cast<const uint4*>(xr[j] + k) : zero;
  };
  uint4 xq[kCache > 0 ? kCache : 1][4][NT], xn[4][NT];
  if (kCache > 0) {
#pragma unroll
    for (int c = 0; c < kCache; ++c)
#pragma unroll
      for (int piece = 0; piece < 4; ++piece)
#pragma unroll
        for (int j = 0; j < NT; ++j) xq[c][piece][j] = c < per_tile ? load_x(c, piece, j) : zero;
  } else if (per_tile > 0) {
#pragma unroll
    for (int piece = 0; piece < 4; ++piece)
#pragma unroll
      for (int j = 0; j < NT; ++j) xn[piece][j] = load_x(0, piece, j);
  }
  const unsigned row_lo = (unsigned)g * 128u, row_hi = (unsigned)(g + 8) * 128u, swz = (unsigned)(g & 7);
  int acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0;

  int n = 0;
  bool gave_up = false;
  auto multiply = [&](int c) {
    request(n + kRing - 1);
    if (!mbar_wait(bars + 8u * (n % kRing), (unsigned)(n / kRing) & 1, p.error_flag, 41)) {
      gave_up = true;
      failed = 1;
      return;
    }
    const unsigned slot = ring + (unsigned)(n % kRing) * kStreamStage;
    uint4 xc[4][NT];
    if (kCache == 0) {
#pragma unroll
      for (int piece = 0; piece < 4; ++piece)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          xc[piece][j] = xn[piece][j];
          xn[piece][j] = load_x(c + 1 < per_tile ? c + 1 : 0, piece, j);      // (every tile meets the same x)
        }
    }
#pragma unroll
    for (int piece = 0; piece < 4; ++piece) {
      const unsigned at = slot + (unsigned)(piece >> 1) * (kStreamStage / 2) + (((unsigned)(2 * t + (piece & 1)) ^ swz) << 4);
      const uint4 wl = lds128(at + row_lo), wh = lds128(at + row_hi);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 xv = kCache > 0 ? xq[c < kCache ? c : 0][piece][j] : xc[piece][j];
        mma_s8(acc[j], wl.x, wh.x, wl.y, wh.y, xv.x, xv.y);
        mma_s8(acc[j], wl.z, wh.z, wl.w, wh.w, xv.z, xv.w);
      }
    }
    __syncwarp();     // every lane has read the stage before lane 0 asks for new contents
    ++n;
  };
  for (int ti = 0; ti < my_tiles; ++ti) {
    const int tile = blockIdx.x + ti * gridDim.x;
    if (kCache > 0) {
#pragma unroll
      for (int c = 0; c < kCache; ++c)
        if (c < per_tile && !gave_up) multiply(c);
    } else {
      for (int c = 0; c < per_tile && !gave_up; ++c) multiply(c);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      partial[warp][g][j * 8 + 2 * t] = acc[j][0];
      partial[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
      partial[warp][g + 8][j * 8 + 2 * t] = acc[j][2];
      partial[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0;
    }
    __syncthreads();
    if (failed) break;        // (uniform: read after the barrier)
    for (int e = threadIdx.x; e < 16 * kCols; e += kWarps * 32) {
      const int r = e % 16, m = e / 16, col = tile * 16 + r;
      if (m >= M || col >= p.N) continue;
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += partial[w][r][m];
      ((T*)p.out)[(size_t)m * p.N + col] = from_float<T>(scaled(sum, p.q_scale[m], p.w_scale[col], (const T*)p.bias, col));
    }
    __syncthreads();          // the partial tiles are free again
  }
  if (gave_up || failed) {
    // Copies that were asked for and never multiplied: a bounded wait for each, so that none lands after the
    // block's shared memory has gone to another block.
    for (int r = n; r < items && r < n + kRing; ++r) mbar_wait(bars + 8u * (r % kRing), (unsigned)(r / kRing) & 1, nullptr, 0);
  }
}

// The same with x's rows quantised by every block for itself, into shared memory: one launch, and no memory but the output's.  x is read
// once, all of it on its way at a time and in registers between its maxima and its rounding (read in turns of 8 K numbers, twice, 32 K
// numbers took 10 us: every trip to L2 costs one, with all SMs at the same lines); so 16 K numbers at most.
constexpr int kFusedNumbers = 1 << 14, kFusedRows = 16;

struct FusedParams {
  const void* x;
  size_t row_stride;
  int inner;                // numbers of a row of x
  bool at_rest;             // w is written by no kernel any more: it is asked for before the kernels ahead are done
};

template <typename T, int NT, int kWarps, int kRing>
__global__ void __launch_bounds__(kWarps * 32)
gemm_int8_fused_kernel(const __grid_constant__ CUtensorMap map_w, const Int8GemmParams p, const FusedParams f) {
  constexpr int kCols = NT * 8, N = Vec16<T>::N, kThreads = kWarps * 32;
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  __shared__ int partial[kWarps][16][kCols + 1];
  __shared__ __align__(8) unsigned long long ring_bars[kWarps * kRing];
  __shared__ int failed;
  __shared__ unsigned tops[kFusedRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int M = p.M, K = f.inner;
  const int tiles = (p.N + 15) / 16, chunks = (p.K + kStreamK - 1) / kStreamK;
  const int per_tile = warp < chunks ? (chunks - warp + kWarps - 1) / kWarps : 0;
  const int my_tiles = (int)blockIdx.x < tiles ? (tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  const int items = my_tiles * per_tile;
  const unsigned ring = base + (unsigned)warp * kRing * kStreamStage;
  const unsigned bars = smem_addr(ring_bars) + (unsigned)warp * kRing * 8;
  // x in 8 bits behind the rings: a row's bytes, zeros up to a whole stage, and 16 more that keep the rows in different banks.
  const unsigned row_bytes = (unsigned)chunks * kStreamK + 16;
  const unsigned xs = base + (unsigned)kWarps * kRing * kStreamStage;
  unsigned char* const xs_at = smem_raw + (xs - smem_addr(smem_raw));

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kRing; ++i) mbar_init(smem_addr(ring_bars) + 8u * i, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < kFusedRows) tops[threadIdx.x] = 0;
  __syncthreads();
  auto request = [&](int n) {
    if (lane != 0 || n >= items) return;
    const int tile = blockIdx.x + (n / per_tile) * gridDim.x, k0 = (warp + (n % per_tile) * kWarps) * kStreamK;
    const unsigned slot = ring + (unsigned)(n % kRing) * kStreamStage, bar = bars + 8u * (n % kRing);
    mbar_expect_tx(bar, kStreamStage);
    tma_load_2d(slot, &map_w, bar, k0, tile * 16);
    tma_load_2d(slot + kStreamStage / 2, &map_w, bar, k0 + 128, tile * 16);
  };
  if (!f.at_rest) grid_dependency_wait();
  for (int n = 0; n < kRing - 1; ++n) request(n);
  grid_launch_dependents();
  grid_dependency_wait();

  // Eight numbers a thread at a time: of row m the eight i, and the thread's next ones without a division.
  constexpr int kHeld = (kFusedNumbers / 8 + kThreads - 1) / kThreads;
  const int eights = (K + 7) / 8, whole = K / 8;
  Vec16<T> held[kHeld][8 / N];
  int m = (int)threadIdx.x / eights, i = (int)threadIdx.x - m * eights;
  const int first_m = m, first_i = i;
  auto next = [&]() {
    i += kThreads;
    while (i >= eights) { i -= eights; ++m; }
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (h * kThreads >= M * eights) break;      // (uniform)
    const T* src = (const T*)f.x + m * f.row_stride + i * 8;
#pragma unroll
    for (int e = 0; e < 8 / N; ++e) {
      if (m < M && i < whole) {
        held[h][e] = load16(src + e * N);
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n) held[h][e].set(n, m < M && i * 8 + e * N + n < K ? to_float(src[e * N + n]) : 0.f);
      }
    }
    next();
  }
  m = first_m;
  i = first_i;
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (h * kThreads >= M * eights) break;
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, abs_bits(held[h][e / N].get(e % N)));
    const int lowest = __shfl_sync(0xffffffffu, m, 0);
    if (lowest == __shfl_sync(0xffffffffu, m, 31)) {        // a warp's eights are of one row but at the rows' ends
      top = warp_max_bits(top);
      if (lane == 0 && m < M) atomicMax(&tops[m], top);
    } else if (m < M) {
      atomicMax(&tops[m], top);
    }
    next();
  }
  for (int z = warp; z < M; z += kWarps)
    for (int k = eights * 8 + lane * 8; k < (int)row_bytes; k += 256) *reinterpret_cast<uint2*>(xs_at + (size_t)z * row_bytes + k) = make_uint2(0, 0);
  __syncthreads();
  m = first_m;
  i = first_i;
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (h * kThreads >= M * eights) break;
    if (m < M) {
      const float s = scale_of(tops[m]);
      const bool plain = scale_plain(s);
      const float inverse = plain ? __frcp_rn(s) : 0.f;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8 / N; ++e) unpack16(held[h][e], v + e * N);
      *reinterpret_cast<uint2*>(xs_at + (size_t)m * row_bytes + i * 8) = make_uint2(quantised4(v, s, inverse, plain), quantised4(v + 4, s, inverse, plain));
    }
    next();
  }
  __syncthreads();

  const unsigned row_lo = (unsigned)g * 128u, row_hi = (unsigned)(g + 8) * 128u, swz = (unsigned)(g & 7);
  unsigned xr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) xr[j] = xs + (unsigned)min(j * 8 + g, M - 1) * row_bytes + (unsigned)(2 * t) * 16;
  int acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0;
  int n = 0;
  bool gave_up = false;
  for (int ti = 0; ti < my_tiles; ++ti) {
    const int tile = blockIdx.x + ti * gridDim.x;
    for (int c = 0; c < per_tile && !gave_up; ++c) {
      request(n + kRing - 1);
      if (!mbar_wait(bars + 8u * (n % kRing), (unsigned)(n / kRing) & 1, p.error_flag, 41)) {
        gave_up = true;
        failed = 1;
        break;
      }
      const unsigned slot = ring + (unsigned)(n % kRing) * kStreamStage, k0 = (unsigned)(warp + c * kWarps) * kStreamK;
#pragma unroll
      for (int piece = 0; piece < 4; ++piece) {
        const unsigned at = slot + (unsigned)(piece >> 1) * (kStreamStage / 2) + (((unsigned)(2 * t + (piece & 1)) ^ swz) << 4);
        const uint4 wl = lds128(at + row_lo), wh = lds128(at + row_hi);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 xv = lds128(xr[j] + k0 + (unsigned)(piece >> 1) * 128u + (unsigned)(piece & 1) * 16u);
          mma_s8(acc[j], wl.x, wh.x, wl.y, wh.y, xv.x, xv.y);
          mma_s8(acc[j], wl.z, wh.z, wl.w, wh.w, xv.z, xv.w);
        }
      }
      __syncwarp();     // every lane has read the stage before lane 0 asks for new contents
      ++n;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      partial[warp][g][j * 8 + 2 * t] = acc[j][0];
      partial[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
      partial[warp][g + 8][j * 8 + 2 * t] = acc[j][2];
      partial[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0;
    }
    __syncthreads();
    if (failed) break;        // (uniform: read after the barrier)
    for (int e = threadIdx.x; e < 16 * kCols; e += kThreads) {
      const int r = e % 16, m = e / 16, col = tile * 16 + r;
      if (m >= M || col >= p.N) continue;
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += partial[w][r][m];
      ((T*)p.out)[(size_t)m * p.N + col] = from_float<T>(scaled(sum, scale_of(tops[m]), p.w_scale[col], (const T*)p.bias, col));
    }
    __syncthreads();          // the partial tiles are free again
  }
  if (gave_up || failed)
    for (int r = n; r < items && r < n + kRing; ++r) mbar_wait(bars + 8u * (r % kRing), (unsigned)(r / kRing) & 1, nullptr, 0);
}

// ------------------------------------------------------------------------------------------------ tensor cores
// Instruction descriptor of kind::i8: 32-bit whole numbers += signed 8-bit x signed 8-bit, both operands K-major.
__device__ __forceinline__ constexpr unsigned i8_desc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned idesc, bool accumulate) {
  const unsigned acc = accumulate ? 1u : 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned idesc, bool accumulate) {
  const unsigned acc = accumulate ? 1u : 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

__device__ __forceinline__ void tmem_load16(unsigned taddr, unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

constexpr int kTileRows = 128;             // rows of w a CTA multiplies
constexpr int kTileK = 128;                // bytes of k a stage: one swizzle row
constexpr int kMmaK = 32;
constexpr unsigned kBytesW = kTileRows * kTileK;
constexpr int kMaxStages = 8;

// ---- cluster: blockIdx.x = tile * splits + split; the cluster's CTAs are the splits of one tile.
constexpr int kClusterThreads = 320;       // loader, issuer, eight warps that empty the accumulator
constexpr size_t kClusterSmem = 200 * 1024;

template <typename T, int splits>
__global__ void __launch_bounds__(kClusterThreads, 1)
gemm_int8_cluster_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Int8GemmParams p) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) unsigned long long bars[2 * kMaxStages + 1];     // full, empty, done
  __shared__ unsigned tmem_slot;
  __shared__ int failed;
  const unsigned bar0 = smem_addr(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  const unsigned done_bar = bar0 + 8u * (2 * kMaxStages);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
  const int tn = tile / p.col_tiles, tm = tile - tn * p.col_tiles;        // (the tiles of the same rows of w run side by side)
  const int n0 = tn * kTileRows, m0 = tm * p.cols;
  const int k_blocks = (p.K + kTileK - 1) / kTileK;
  const int kb_lo = (int)((long)k_blocks * split / splits), kb_hi = (int)((long)k_blocks * (split + 1) / splits);
  const unsigned stage_bytes = kBytesW + (unsigned)p.cols * kTileK;

  if (threadIdx.x == 0) {
    prefetch_map(&map_w);
    prefetch_map(&map_x);
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const unsigned tmem = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // The weights of the first stages wait for nobody; x comes from the kernel ahead.
      const int early = min(p.stages, kb_hi - kb_lo);
      for (int i = 0; i < early; ++i) {
        mbar_expect_tx(full_bar(i), stage_bytes);
        tma_load_2d(base + i * stage_bytes, &map_w, full_bar(i), (kb_lo + i) * kTileK, n0);
      }
      grid_launch_dependents();
      grid_dependency_wait();
      for (int i = 0; i < early; ++i) tma_load_2d(base + i * stage_bytes + kBytesW, &map_x, full_bar(i), (kb_lo + i) * kTileK, m0);
      int stage = 0, asked = early;
      unsigned phase = 1;
      for (int kb = kb_lo + early; kb < kb_hi; ++kb) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1, p.error_flag, 42)) { failed = 1; break; }
        mbar_expect_tx(full_bar(stage), stage_bytes);
        tma_load_2d(base + stage * stage_bytes, &map_w, full_bar(stage), kb * kTileK, n0);
        tma_load_2d(base + stage * stage_bytes + kBytesW, &map_x, full_bar(stage), kb * kTileK, m0);
        ++asked;
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      // What was asked for lands before the block ends, also where a wait gave up (the issuer's, say).
      for (int i = max(0, asked - p.stages); i < asked; ++i) mbar_wait(full_bar(i % p.stages), (unsigned)(i / p.stages) & 1, nullptr, 0);
    }
  } else if (warp == 1) {
    const unsigned idesc = i8_desc(kTileRows, p.cols);
    const unsigned long long first = umma_desc(base);
    int stage = 0;
    unsigned phase = 0;
    bool ok = true;
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
      if (!warp_wait(full_bar(stage), phase, p.error_flag, 43)) { ok = false; break; }
      tcgen05_fence_after();
      const unsigned long long a = first + (unsigned long long)((stage * stage_bytes) >> 4), b = a + (kBytesW >> 4);
      if (elected()) {
#pragma unroll
        for (int k = 0; k < kTileK / kMmaK; ++k)
          umma_i8(tmem, a + (unsigned long long)((k * kMmaK) >> 4), b + (unsigned long long)((k * kMmaK) >> 4), idesc, kb > kb_lo || k > 0);
        umma_commit(empty_bar(stage));
      }
      __syncwarp();
      if (++stage == p.stages) { stage = 0; phase ^= 1; }
    }
    if (elected()) {
      if (!ok) failed = 1;
      umma_commit(done_bar);
    }
  }
  __syncwarp();     // (lanes that went ahead would wait below in the way of their own warp's loader or issuer: 56 us instead of 16)
  // Everybody waits for the products: the stages' memory then takes the sums, a column (a row of x) behind the other.
  bool ok = mbar_wait(done_bar, 0, p.error_flag, 44);
  grid_dependency_wait();       // (the scales of x come from the kernel ahead as well)
  tcgen05_fence_after();
  __syncthreads();
  ok = ok && failed == 0;
  int* sums = reinterpret_cast<int*>(smem_raw + (base - smem_addr(smem_raw)));       // [cols][128]
  if (warp >= 2 && ok) {
    // Two warps share a quarter of the lanes and take 16 columns in turn, two loads on their way.
    const int quarter = warp & 3;
    const unsigned from = tmem + ((unsigned)(quarter * 32) << 16);
    int* const to = sums + quarter * 32 + lane;
    for (int c = (warp - 2) / 4 * 16; c < p.cols; c += 64) {
      unsigned r[2][16];
      const bool both = c + 32 < p.cols;
      tmem_load16(from + (unsigned)c, r[0]);
      if (both) tmem_load16(from + (unsigned)(c + 32), r[1]);
      tmem_load_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) to[(c + j) * kTileRows] = (int)r[0][j];
      if (both) {
#pragma unroll
        for (int j = 0; j < 16; ++j) to[(c + 32 + j) * kTileRows] = (int)r[1][j];
      }
    }
  }
  tcgen05_fence_before();
  if (splits > 1) cluster_sync_all();     // (release and acquire: every CTA's sums are there)
  else __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
  }
  // A warp a column at a time, four rows of w a lane; the cluster's CTAs share the columns.
  const int live = min(p.cols, p.M - m0);
  const int n = n0 + lane * 4;
  float s_w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s_w[i] = n + i < p.N ? p.w_scale[n + i] : 0.f;
  constexpr int kAtOnce = 4, kWarpsHere = kClusterThreads / 32;      // columns on their way: a remote load takes about a microsecond
  if (ok)
    for (int c0 = split + warp * splits; c0 < live; c0 += kAtOnce * splits * kWarpsHere) {
      int4 part[kAtOnce][splits];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int c = c0 + i * splits * kWarpsHere;
        if (c >= live) break;
        const unsigned at = smem_addr(sums + c * kTileRows + lane * 4);
#pragma unroll
        for (int s = 0; s < splits; ++s) {
          if (splits == 1) {
            part[i][s] = *reinterpret_cast<const int4*>(sums + c * kTileRows + lane * 4);
          } else {
            unsigned remote;
            int4& v = part[i][s];
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(s));
            asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
      const int c = c0 + i * splits * kWarpsHere;
      if (c >= live) break;
      int4 sum = part[i][0];
#pragma unroll
      for (int s = 1; s < splits; ++s) {
        sum.x += part[i][s].x; sum.y += part[i][s].y; sum.z += part[i][s].z; sum.w += part[i][s].w;
      }
      const float s_x = p.q_scale[m0 + c];
      T* dst = (T*)p.out + (size_t)(m0 + c) * p.N + n;
      const int all[4] = {sum.x, sum.y, sum.z, sum.w};
      if (n + 4 <= p.N && p.N % 4 == 0) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = scaled(all[i], s_x, s_w[i], (const T*)p.bias, n + i);
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
          *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.N) dst[i] = from_float<T>(scaled(all[i], s_x, s_w[i], (const T*)p.bias, n + i));
      }
      }
    }
  if (splits > 1) cluster_sync_all();     // nobody leaves while another reads its sums
}

// ---- pair: a pair of CTAs (cta_group::2) on a tile of 256 rows of w by p.cols rows of x, each CTA with 128 rows of w and half the rows
// of x in shared memory and its 128 rows of the sums in tensor memory, two tiles' worth of them.
constexpr int kPairStages = 6;
constexpr int kPairWarps = 12;             // that empty the accumulators
constexpr int kPairThreads = 64 + 32 * kPairWarps;
constexpr int kTurnRow = 40;               // bfloat16 of a row being turned: 32 and the padding that keeps 16-byte alignment
constexpr unsigned kPairStage = kBytesW + 128 * kTileK;
constexpr size_t kPairSmem = 1024 + kPairStages * kPairStage + kPairWarps * 32 * kTurnRow * 2 + 8 * (2 * kPairStages + 5);

// Tiles are walked in bands of eight tiles of w, x's tiles side by side inside a band, so that the pairs running at the same time
// share a few tiles of either (which then come from L2).
__device__ __forceinline__ void pair_tile(int tile, int tiles_n, int tiles_m, int& tn, int& tm) {
  constexpr int kBand = 8;
  const int per_band = kBand * tiles_m;
  const int band = tile / per_band, in_band = tile - band * per_band;
  const int rows = min(kBand, tiles_n - band * kBand);
  tm = in_band / rows;
  tn = band * kBand + in_band % rows;
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Int8GemmParams p) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const unsigned turn = base + kPairStages * kPairStage, bars = turn + kPairWarps * 32 * kTurnRow * 2;
  auto full_bar = [&](int s) { return bars + 8u * s; };                       // waited on in the leader only
  auto empty_bar = [&](int s) { return bars + 8u * (kPairStages + s); };      // signalled in both CTAs
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kPairStages + b); };         // signalled in both CTAs
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kPairStages + 2 + b); };    // the leader's: both CTAs' warps arrive
  const unsigned drained_bar = bars + 8u * (2 * kPairStages + 4);                       // signalled in both CTAs
  __shared__ unsigned tmem_slot;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = cluster_cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles_n = (p.N + 2 * kTileRows - 1) / (2 * kTileRows), num_tiles = tiles_n * p.col_tiles;
  const int k_blocks = (p.K + kTileK - 1) / kTileK;
  const unsigned tile_bytes = kBytesW + (unsigned)(p.cols / 2) * kTileK;

  if (threadIdx.x == 0) {
    prefetch_map(&map_w);
    prefetch_map(&map_x);
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 2 * kPairWarps);
    }
    mbar_init(drained_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {   // the same warp in both CTAs: the allocation is made for the pair
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  cluster_sync_all();       // both CTAs' barriers exist before either signals the other
  const unsigned tmem = tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, asked = 0;
      unsigned phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += pairs) {
        int tn, tm;
        pair_tile(tile, tiles_n, p.col_tiles, tn, tm);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, p.error_flag, 45)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * tile_bytes);   // the bytes of both CTAs
          const unsigned a = base + stage * kPairStage;
          tma_load_2d_pair(a, &map_w, full_bar(stage), kb * kTileK, tn * 2 * kTileRows + (int)rank * kTileRows);
          tma_load_2d_pair(a + kBytesW, &map_x, full_bar(stage), kb * kTileK, tm * p.cols + (int)rank * (p.cols / 2));
          ++asked;
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      // What either CTA asked for lands before the pair ends, also where a wait gave up.
      if (rank == 0)
        for (int i = max(0, asked - kPairStages); i < asked; ++i) mbar_wait(full_bar(i % kPairStages), (unsigned)(i / kPairStages) & 1, nullptr, 0);
    }
  } else if (warp == 1) {
    // The whole warp goes along and one of its lanes issues: a lane that is alone in a branch takes some 100 cycles a product for it, as much
    // as the product (8,192 x 4,096 x 14,336: 340 us, 322 with this).
    if (rank == 0) {
      const unsigned idesc = i8_desc(2 * kTileRows, p.cols);
      const unsigned long long first = umma_desc(base);
      int stage = 0, local = 0;
      unsigned phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < num_tiles; tile += pairs, ++local) {
        const int buf = local & 1;
        if (!warp_wait(acc_empty_bar(buf), ((unsigned)(local >> 1) & 1) ^ 1, p.error_flag, 46)) { ok = false; break; }
        tcgen05_fence_after();
        const unsigned acc = tmem + (unsigned)(buf * 256);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!warp_wait(full_bar(stage), phase, p.error_flag, 47)) { ok = false; break; }
          tcgen05_fence_after();
          const unsigned long long a = first + (unsigned long long)((stage * kPairStage) >> 4), b = a + (kBytesW >> 4);
          if (elected()) {
#pragma unroll
            for (int k = 0; k < kTileK / kMmaK; ++k)
              umma_i8_pair(acc, a + (unsigned long long)((k * kMmaK) >> 4), b + (unsigned long long)((k * kMmaK) >> 4), idesc, kb > 0 || k > 0);
            umma_commit_pair(empty_bar(stage));
            if (kb + 1 == k_blocks) umma_commit_pair(acc_full_bar(buf));
          }
          __syncwarp();
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) {        // products that are under way still are done before tensor memory goes back
        if (elected()) umma_commit_pair(drained_bar);
        warp_wait(drained_bar, 0, nullptr, 0);
      }
    }
  } else {
    // A warp may read the 32 lanes of tensor memory that its number modulo four names (32 rows of w); the warps that share a quarter
    // take 32 rows of x in turn.
    const int quarter = warp & 3, which = (warp - 2) >> 2;
    bf16* const mine = reinterpret_cast<bf16*>(smem_raw + (turn - smem_addr(smem_raw))) + (warp - 2) * 32 * kTurnRow;
    int local = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < num_tiles; tile += pairs, ++local) {
      int tn, tm;
      pair_tile(tile, tiles_n, p.col_tiles, tn, tm);
      const int buf = local & 1;
      const int f0 = tn * 2 * kTileRows + (int)rank * kTileRows + quarter * 32, n = f0 + lane;       // this lane's row of w
      const float s_w = n < p.N ? p.w_scale[n] : 0.f;
      if (!mbar_wait(acc_full_bar(buf), (unsigned)(local >> 1) & 1, p.error_flag, 48)) { ok = false; break; }
      tcgen05_fence_after();
      const unsigned taddr = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(buf * 256);
      const int live = min(p.cols, p.M - tm * p.cols);
#pragma unroll 1
      for (int c = which * 32; c < live; c += 8 * kPairWarps) {
        unsigned r[32];
        __syncwarp();                       // the load below is a warp-wide instruction; and `mine` has been read
        tmem_load32(taddr + c, r);
        const int m = tm * p.cols + c;      // the first of these rows of x
        const bool stores = c + lane < live;
        const float s_x = stores ? p.q_scale[m + lane] : 0.f;
        tmem_load_wait();
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float v = scaled((int)r[j], __shfl_sync(0xffffffffu, s_x, j), s_w, (const T*)(n < p.N ? p.bias : nullptr), n);
            if (c + j < live && n < p.N) ((float*)p.out)[(size_t)(m + j) * p.N + n] = v;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            mine[j * kTurnRow + lane] = __float2bfloat16_rn(
                scaled((int)r[j], __shfl_sync(0xffffffffu, s_x, j), s_w, (const T*)(n < p.N ? p.bias : nullptr), n));
          __syncwarp();
          // A row is a lane's where rows begin at 16 bytes.  Where they do not, a row goes out whole at a time, in pairs of numbers where
          // they begin at four: its lanes' stores lie side by side (7,876 x 640 x 2,842: 244 us with a row a lane, 44 with this).
          if (p.N % 8 == 0) {
            if (stores) {
              bf16* dst = (bf16*)p.out + (size_t)(m + lane) * p.N + f0;
              const bf16* src = mine + lane * kTurnRow;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (f0 + e * 8 < p.N) *reinterpret_cast<uint4*>(dst + e * 8) = *reinterpret_cast<const uint4*>(src + e * 8);
            }
          } else if (p.N % 2 == 0) {
            const int col = (lane & 15) * 2;
            if (f0 + col < p.N) {
#pragma unroll 8
              for (int j = lane >> 4; j < 32; j += 2)
                if (c + j < live)
                  *reinterpret_cast<unsigned*>((bf16*)p.out + (size_t)(m + j) * p.N + f0 + col) = *reinterpret_cast<const unsigned*>(mine + j * kTurnRow + col);
            }
          } else if (n < p.N) {
#pragma unroll 8
            for (int j = 0; j < 32; ++j)
              if (c + j < live) ((bf16*)p.out)[(size_t)(m + j) * p.N + n] = mine[j * kTurnRow + lane];
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(acc_empty_bar(buf));
    }
  }
  tcgen05_fence_before();
  cluster_sync_all();        // neither CTA leaves, nor frees tensor memory, while the other may still use it
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ launches
// A [rows, K] matrix of bytes as a 2-D map with boxes of 128 x box_rows and the 128-byte swizzle; what lies outside reads as zero.
static bool byte_map(CUtensorMap* map, const void* ptr, int rows, int K, int stride, int box_rows) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {(cuuint32_t)kTileK, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int device_sms() {
  static int sms = 0;
  if (!sms) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms < 1)
      sms = 148;
  }
  return sms;
}

static bool streams(int M, int N, int sms);

template <typename T, int NT, int kWarps, int kRing, int kCache>
static int launch_stream(const CUtensorMap& map, const Int8GemmParams& p, int grid, cudaStream_t stream) {
  constexpr size_t smem = (size_t)kWarps * kRing * kStreamStage + 1024;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_stream_kernel<T, NT, kWarps, kRing, kCache>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return (int)launch_maybe_early(pdl_mode() >= 1, gemm_int8_stream_kernel<T, NT, kWarps, kRing, kCache>, dim3(grid), dim3(kWarps * 32), smem, stream, map, p);
}

template <typename T, int NT>
static int stream_product(const CUtensorMap& map, const Int8GemmParams& p, cudaStream_t stream) {
  const int tiles = (p.N + 15) / 16, sms = device_sms(), chunks = (p.K + kStreamK - 1) / kStreamK;
  constexpr int kKeep = NT == 1 ? 3 : NT == 2 ? 1 : 0;          // stages whose x fits a warp's registers
  if (tiles <= 2 * sms || NT == 4) {
    if (kKeep > 0 && chunks <= 8 * kKeep) return launch_stream<T, NT, 8, 3, kKeep>(map, p, tiles, stream);
    return launch_stream<T, NT, 8, 3, 0>(map, p, tiles <= 2 * sms ? tiles : sms, stream);
  }
  if constexpr (NT == 4) return LI_ERR_UNSUPPORTED;      // (not reached)
  else if (kKeep > 0 && chunks <= 6 * kKeep) return launch_stream<T, NT, 6, 3, kKeep>(map, p, 2 * sms, stream);
  else return launch_stream<T, NT, 6, 3, 0>(map, p, 2 * sms, stream);
}

template <typename T, int NT, int kWarps, int kRing>
static int launch_fused(const CUtensorMap& map, const Int8GemmParams& p, const FusedParams& f, int grid, cudaStream_t stream) {
  constexpr size_t rings = (size_t)kWarps * kRing * kStreamStage + 1024;
  constexpr size_t most = rings + kFusedNumbers + kFusedRows * (kStreamK + 16);
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_fused_kernel<T, NT, kWarps, kRing>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const size_t smem = rings + (size_t)p.M * ((size_t)(p.K + kStreamK - 1) / kStreamK * kStreamK + 16);
  return (int)launch_maybe_early(pdl_mode() >= 1, gemm_int8_fused_kernel<T, NT, kWarps, kRing>, dim3(grid), dim3(kWarps * 32), smem, stream, map, p, f);
}

// Whether a product can go without a kernel ahead of it that quantises x.
static bool fuses(const Int8GemmParams& p, const FusedParams& f, size_t size) {
  return p.M <= kFusedRows && (long)p.M * p.K <= kFusedNumbers && aligned16(f.x) && f.row_stride * size % 16 == 0 && streams(p.M, p.N, device_sms());
}

template <typename T>
static int fused_product(const Int8GemmParams& p, const FusedParams& f, const void* w, cudaStream_t stream) {
  CUtensorMap map;
  if (!byte_map(&map, w, p.N, p.K, p.K, 16)) return LI_ERR_UNSUPPORTED;
  const int tiles = (p.N + 15) / 16, sms = device_sms();
  // A weight of few tiles has a block of eight warps for each; more tiles go to blocks that walk them, two an SM.
  if (tiles <= sms) return p.M <= 8 ? launch_fused<T, 1, 8, 3>(map, p, f, tiles, stream) : launch_fused<T, 2, 8, 3>(map, p, f, tiles, stream);
  return p.M <= 8 ? launch_fused<T, 1, 6, 3>(map, p, f, min(tiles, 2 * sms), stream) : launch_fused<T, 2, 6, 3>(map, p, f, min(tiles, 2 * sms), stream);
}

template <typename T, int splits>
static int cluster_product(const CUtensorMap& mw, const CUtensorMap& mx, const Int8GemmParams& p, int tiles, cudaStream_t stream) {
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_cluster_kernel<T, splits>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kClusterSmem);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(tiles * splits);
  config.blockDim = dim3(kClusterThreads);
  config.dynamicSmemBytes = kClusterSmem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = splits;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = pdl_enabled(0) ? 2 : 1;
  return (int)cudaLaunchKernelEx(&config, gemm_int8_cluster_kernel<T, splits>, mw, mx, p);
}

template <typename T>
static int pair_product(const CUtensorMap& mw, const CUtensorMap& mx, const Int8GemmParams& p, int tiles, cudaStream_t stream) {
  static_assert(kPairSmem <= 232448 - 64, "more shared memory than a block may have");
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(gemm_int8_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  const int sms = device_sms();
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(2 * (tiles < sms / 2 ? tiles : sms / 2));
  config.blockDim = dim3(kPairThreads);
  config.dynamicSmemBytes = kPairSmem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = 2;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = pdl_enabled(0) ? 2 : 1;
  return (int)cudaLaunchKernelEx(&config, gemm_int8_pair_kernel<T>, mw, mx, p);
}

// Few rows of x stream w.  Up to eight are one tile of eight; up to 32 more of them share its reads, but read x again for every tile of
// w, and the tensor cores' fixed 3 us pay for themselves the sooner, the more tiles there are.  Measured on B200, stream and cluster,
// microseconds with the quantisation: 8 rows of 2,048 x 2,048 4.3 and 6.5, 4,096 x 14,336 13.9 and 16.0; 16 rows of 8,192 x 2,048 8.9 and 10.9, 4,096 x
// 4,096 8.1 and 9.5, 2,048 x 16,384 14.1 and 11.7; 32 rows of 2,048 x 2,048 5.9 and 6.7, 8,192 x 2,048 11.0 and 10.9, 4,096 x 4,096 12.2 and 9.6.
static bool streams(int M, int N, int sms) {
  const int tiles = (N + 15) / 16;
  return M <= 8 || (M <= 16 && tiles <= 2 * sms) || (M <= 32 && tiles <= sms);
}

template <typename T>
static int product(Int8GemmParams p, const void* w, cudaStream_t stream) {
  const int sms = device_sms();
  CUtensorMap mw, mx;
  if (streams(p.M, p.N, sms)) {
    if (!byte_map(&mw, w, p.N, p.K, p.K, 16)) return LI_ERR_UNSUPPORTED;
    return p.M <= 8 ? stream_product<T, 1>(mw, p, stream) : p.M <= 16 ? stream_product<T, 2>(mw, p, stream) : stream_product<T, 4>(mw, p, stream);
  }
  // Tiles of 128 rows of w, and x's rows in as few tiles of at most 256 as there can be, equal ones.
  const int row_tiles = (p.N + kTileRows - 1) / kTileRows;
  p.col_tiles = (p.M + 255) / 256;
  if (row_tiles * p.col_tiles <= sms) {
    // Where that leaves SMs idle that would not be enough to share tiles' k, smaller tiles (1,093 x 2,096 x 2,604: 105 tiles 17.4 us, 147 15.6).
    if (2 * row_tiles * p.col_tiles > sms) p.col_tiles = sms / row_tiles;
    p.cols = ((p.M + p.col_tiles - 1) / p.col_tiles + 15) / 16 * 16;
    p.col_tiles = (p.M + p.cols - 1) / p.cols;
    const unsigned stage = kBytesW + (unsigned)p.cols * kTileK;
    p.stages = (int)((kClusterSmem - 1024) / stage);
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    const int tiles = row_tiles * p.col_tiles, k_blocks = (p.K + kTileK - 1) / kTileK;
    int splits = 1;
    // As many CTAs share a tile's k as all run at once, two steps of k each at least.  (Clusters of eight of them, 200 KB each, do not: 128 in
    // such clusters took two rounds, 64 rows of 8,192 x 2,048 15.8 us, with four 11.7.)
    while (splits < 4 && 2 * splits * tiles <= sms && 4 * splits <= k_blocks) splits *= 2;
    if (!byte_map(&mw, w, p.N, p.K, p.K, kTileRows) || !byte_map(&mx, p.q, p.M, p.K, p.q_stride, p.cols)) return LI_ERR_UNSUPPORTED;
    return splits == 1 ? cluster_product<T, 1>(mw, mx, p, tiles, stream) : splits == 2 ? cluster_product<T, 2>(mw, mx, p, tiles, stream)
                                                                                               : cluster_product<T, 4>(mw, mx, p, tiles, stream);
  }
  // The pairs take the tiles in rounds; of all sizes of a tile, that with the least rounds x (rows of x + 64), the 64 for what a tile costs
  // whatever it is wide (467 x 3,600 x 11,728: two rounds of 256 wide 32 us, two of 160 30).
  const int w_tiles = (p.N + 2 * kTileRows - 1) / (2 * kTileRows), pairs = sms / 2;
  long best = -1;
  for (int cols = 256; cols >= 128; cols -= 32) {
    const long rounds = ((long)w_tiles * ((p.M + cols - 1) / cols) + pairs - 1) / pairs, cost = rounds * (cols + 64);
    if (best < 0 || cost < best) {
      best = cost;
      p.cols = cols;
    }
  }
  p.col_tiles = (p.M + p.cols - 1) / p.cols;
  if (!byte_map(&mw, w, p.N, p.K, p.K, kTileRows) || !byte_map(&mx, p.q, p.M, p.K, p.q_stride, p.cols / 2)) return LI_ERR_UNSUPPORTED;
  const long tiles = (long)((p.N + 2 * kTileRows - 1) / (2 * kTileRows)) * p.col_tiles;
  if (tiles > 0x3fffffffL) return LI_ERR_UNSUPPORTED;
  return pair_product<T>(mw, mx, p, (int)tiles, stream);
}

}  // namespace li

using namespace li;

struct QuantiseRowsArgs {
  long long dtype;          // of x
  const void* x;
  long long row_stride;
  void* q;                  // [M][q_stride], zeros from K on
  long long q_stride;       // a multiple of 16, at least K
  float* scale;
  long long M, K;
  cudaStream_t stream;
};

LI_EXPORT int li_quantise_rows(const QuantiseRowsArgs* a) {
  if (a->M == 0) return 0;
  if (a->K < 1 || a->q_stride < a->K || a->q_stride % 16) return LI_ERR_UNSUPPORTED;
  if (!aligned16(a->q)) return LI_ERR_ALIGNMENT;
  return a->dtype == kFloat32 ? quantise_rows<float>(a->x, a->row_stride, a->q, (int)a->q_stride, a->scale, (int)a->M, (int)a->K, a->stream)
                              : quantise_rows<bf16>(a->x, a->row_stride, a->q, (int)a->q_stride, a->scale, (int)a->M, (int)a->K, a->stream);
}

struct LinearInt8Args {
  QuantiseRowsArgs rows;    // x [M, K], its place in 8 bits q [M][at least padded] and its scales (the caller's, 16-byte aligned; q null: none)
  const void* w;            // [N][padded]
  long long padded;
  const float* w_scale;
  const void* bias;         // of x's type, or null
  void* out;                // [M][N] of x's type
  long long N;
  int* error_flag;
  long long at_rest;        // no kernel writes w any more
};

#define LI_NEEDS_PLACE 100003

// Multiplies by w, x quantised on the way; padded: a multiple of 16, at least K and at most 131,072.  Without a place for x in 8 bits, only where the
// product needs none; LI_NEEDS_PLACE says that it does, and nothing has been launched.  error_flag (device int, zero): the number of a
// bounded wait that gave up (41 stream, 42 to 44 cluster, 45 to 48 pair); the output is then not to be trusted.
LI_EXPORT int li_linear_int8(const LinearInt8Args* a) {
  const QuantiseRowsArgs& r = a->rows;
  if (r.M == 0 || a->N == 0) return 0;
  if (r.K < 1 || a->padded < r.K || a->padded % 16 || a->padded > 131072 || r.q_stride < a->padded || r.q_stride % 16 || r.M > 0x7fffffffL || a->N > 0x7fffffffL) return LI_ERR_UNSUPPORTED;
  if (!aligned16(a->w) || !aligned16(a->out)) return LI_ERR_ALIGNMENT;
  Int8GemmParams p{(const signed char*)r.q, r.scale, a->w_scale, a->bias, a->out, (int)r.M, (int)a->N, (int)a->padded, (int)r.q_stride, a->error_flag, 0, 0, 0};
  if (r.q == nullptr) {
    const FusedParams f{r.x, (size_t)r.row_stride, (int)r.K, a->at_rest != 0};
    if (!fuses(p, f, r.dtype == kFloat32 ? 4 : 2)) return LI_NEEDS_PLACE;
    return r.dtype == kFloat32 ? fused_product<float>(p, f, a->w, r.stream) : fused_product<bf16>(p, f, a->w, r.stream);
  }
  const int code = li_quantise_rows(&r);
  if (code) return code;
  return r.dtype == kFloat32 ? product<float>(p, a->w, r.stream) : product<bf16>(p, a->w, r.stream);
}
