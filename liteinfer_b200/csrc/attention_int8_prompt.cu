// Attention of portions of prompts over a cache held in 8 bits, on the fifth-generation tensor cores (head sizes 64 and 128, pages of a
// multiple of 16 tokens).
//
// Two kernels.  The first (expand) lays out what the portions can see: keys as whole numbers in bfloat16 (in halves next to queries of 32
// bits) and values as whole numbers in halves, all exact, [portion][kv head][token][dimension], and for every page and head what its scales make of a score and of
// a weight.  It reads a byte and writes two, once, where the second reads the tile once for every 128 / group queries; it knows no block
// table any more.
//
// The second (prompt) has the scales in its softmax:
//
//   w_j = exp2(f_g s_j + d_g - r),   f_g = scale log2(e) s_k,  d_g = log2 s_v  of the page of key j,  s_j = q . k_j with whole k_j,
//   out = sum_j w_j v_j / sum_g 2^-d_g sum_{j in g} w_j     with whole v_j,
//
// so a page's scales cost one factor and one summand in the multiply-add that a score goes through anyway, and one product a page for
// the denominator.  Rounded are only the weights (to halves, 11 bits; the reference r keeps a row's largest between 2^6 and 2^14) and the
// result: with keys, weights and values in bfloat16 instead, the error was 2.7 times what the result's own rounding makes (0.0046
// against 0.0017 for 4,096 queries behind 1,000, 32 heads on 8 of 128).  A page of zeros (s_v = 0) counts as one of scale 2^-60.
// Of 32 bits, queries and weights go as the sum of two halves each, s_v is a factor behind the exponential, and every step's sums are added to
// a second accumulator in 32 bits.
//
// A block holds two tiles of 128 rows (a row: a query and a head of the group) of which each walks the keys 128 at a time: S = Q K^T into
// tensor memory, the softmax, whose weights go over S, O += P V.  Tensor memory is full with two S and two O of head size 128, so a tile's
// chain (softmax, P V, next S) has nothing to overlap with but the other tile's: one warp issues both tiles' products in turn, which
// puts them half a period apart.  What bounds it is that chain, some 3,500 cycles of 128 keys of two tiles of which the tensor
// cores work 2,000 (4,096 queries behind 1,000 as above: 209 us and 10 for the pages, of 222 and 11 with the pages read back to
// bfloat16; the products alone would take 120).  What was measured on the way, whole calls of that case:
//   64 keys a tile, S twice (nothing waits for S)      241 us: a product of 64 keys takes as long as one of 128
//   a thread a row                                     260;  two threads a row, a half of the keys each, 236
//   a quarter (an eighth) of the exponentials as a polynomial on the multiply-add units: 236 (221) of 225 with none
//   queries fetched by TMA instead of by their threads: 5,000 cycles less a block.
#include "int8.cuh"
#include "tcgen05.cuh"

namespace li {

// ------------------------------------------------------------------------------------------------ expand
struct ExpandParams {
  const signed char* pool[2];
  const float* scale[2];
  const int* block_table;
  int table_stride;
  const int* query_start_loc;
  const int* context_lens;
  const int* row_index;     // optional: batch row of each portion (negative: none)
  int window, keep_first;
  float score;              // |scale| * log2(e), or with capped scores |scale| / cap
  unsigned flip;            // what turns two keys' signs where the scale is negative (the softmax wants factors that are not), else 0
  uint4* out[2];            // [rows][kv_heads][blocks * page_size][head_dim] of 16 bits
  float4* runs;             // [rows][kv_heads][blocks * page_size / 16]: f, lv, 2^-lv, 2^lv of 16 tokens
  int blocks, kv_heads, head_dim, page_size, num_pages;
  bool half_keys;           // keys in halves as well
};

__device__ __forceinline__ unsigned sub_f16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ unsigned sub_bf16x2(unsigned a, unsigned b) {
  unsigned r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The low two bytes of a word as two halves: below the byte 0x64, with the sign bit turned, a byte b is 1024 + (b + 128).
__device__ __forceinline__ unsigned as_halves(unsigned w) { return sub_f16x2(__byte_perm(w, 0, 0x4140) ^ 0x64806480u, 0x64806480u); }
// ... as two bfloat16: 128 + (the seven low bits), less 128 or, where the sign bit makes the exponent one larger, 256.
__device__ __forceinline__ unsigned as_bfloats(unsigned w) {
  const unsigned spread = __byte_perm(w, 0, 0x4140);
  return sub_bf16x2((spread & 0x007f007fu) | 0x43004300u, (spread & 0x00800080u) | 0x43004300u);
}

__global__ void __launch_bounds__(256) expand_pages_int8_kernel(const ExpandParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int b = blockIdx.x, which = blockIdx.y & 1, part = blockIdx.y >> 1, parts = gridDim.y >> 1, i = blockIdx.z;
  const int row = p.row_index != nullptr ? p.row_index[i] : i;
  if (row < 0) return;
  const int len = p.context_lens[row], begin = p.query_start_loc[row], end = p.query_start_loc[row + 1], first = b * p.page_size;
  int page = p.block_table[(size_t)row * p.table_stride + b];
  const int pos = len - (end - begin);       // of the first query
  if (first >= len) return;
  if (first + p.page_size <= first_visible(pos, p.window) && first >= p.keep_first) return;      // nobody looks there
  if (page >= p.num_pages) page = -1;
  const size_t from = (size_t)max(page, 0) * p.kv_heads;
  if (blockIdx.y == 0 && threadIdx.x < p.kv_heads) {
    const float k = page >= 0 ? p.scale[0][from + threadIdx.x] : 0.f, v = page >= 0 ? p.scale[1][from + threadIdx.x] : 0.f;
    // (2^-90 at least, or the denominator's 2^-lv could pass float32's range; a NaN stays one)
    const float log2_v = log2f(v), lv = v == 0.f ? -60.f : log2_v < -90.f ? -90.f : log2_v;
    const int runs = p.page_size / 16;
    float4* out = p.runs + (((size_t)i * p.kv_heads + threadIdx.x) * p.blocks + b) * runs;
    // (tokens of no page weigh nothing)
    for (int g = 0; g < runs; ++g)
      out[g] = page < 0 ? make_float4(0.f, -INFINITY, 0.f, 0.f) : make_float4(k * p.score, lv, exp2f(-lv), lv == log2_v ? v : exp2f(lv));
  }
  const int vectors = p.page_size * p.head_dim / 16;      // of a head
  const bool halves = which || p.half_keys;
  const unsigned flip = which ? 0u : p.flip;
  const uint4* in = reinterpret_cast<const uint4*>(p.pool[which]) + from * vectors;
#pragma unroll 4
  for (int v = part * (int)blockDim.x + threadIdx.x; v < p.kv_heads * vectors; v += parts * (int)blockDim.x) {
    const int h = v / vectors;
    const uint4 raw = page >= 0 ? in[v] : make_uint4(0, 0, 0, 0);
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
    unsigned r[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[2 * e] = (halves ? as_halves(w[e]) : as_bfloats(w[e])) ^ flip;
      r[2 * e + 1] = (halves ? as_halves(w[e] >> 16) : as_bfloats(w[e] >> 16)) ^ flip;
    }
    uint4* out = p.out[which] + ((((size_t)i * p.kv_heads + h) * p.blocks + b) * vectors + (v - h * vectors)) * 2;
    out[0] = make_uint4(r[0], r[1], r[2], r[3]);
    out[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// Queries of 32 bits as the sum of two halves, h + l = q / factor with the largest of a head's numbers between 2^10 and 2^11: 22 bits of each
// number stay (and 2^-36 of the largest).  A warp a (token, head); out: all h, then all l, [tokens][heads][head_dim] each.
__global__ void __launch_bounds__(256)
split_queries_kernel(const float* __restrict__ q, int row_stride, __half* __restrict__ out, float* __restrict__ factors, int tokens, int heads, int head_dim) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int item = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= tokens * heads) return;
  const float* from = q + (size_t)(item / heads) * row_stride + (size_t)(item % heads) * head_dim;
  float2 v[2];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = i * 64 < head_dim ? *reinterpret_cast<const float2*>(from + i * 64 + lane * 2) : make_float2(0.f, 0.f);
    top = max(top, max(abs_bits(v[i].x), abs_bits(v[i].y)));
  }
  top = warp_max_bits(top);
  const int exponent = min(max((int)(top >> 23), 24), 254);       // (of zeros and numbers below 2^-103: as if 2^-103 were the largest)
  const float factor = top >= 0x7f800000u ? NAN : __uint_as_float((unsigned)(exponent - 10) << 23);
  const float inverse = 1.f / factor;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (i * 64 < head_dim) {
      const float2 x = make_float2(v[i].x * inverse, v[i].y * inverse);
      const __half2 h = __floats2half2_rn(x.x, x.y);
      const float2 back = __half22float2(h);
      const size_t at = (size_t)item * head_dim + i * 64 + lane * 2;
      *reinterpret_cast<__half2*>(out + at) = h;
      *reinterpret_cast<__half2*>(out + (size_t)tokens * heads * head_dim + at) = __floats2half2_rn(x.x - back.x, x.y - back.y);
    }
  if (lane == 0) factors[item] = factor;
}

// ------------------------------------------------------------------------------------------------ attention
constexpr int kRows = 128;       // rows (query token x head in group) per tile
constexpr int kKeys = 128;       // keys per tile
constexpr int kRuns = kKeys / 16;
constexpr float kHeadroom = 6.f;        // a row's largest weight is 2^kHeadroom when its reference moves,
constexpr float kLargest = 16384.f;     // which it does when the weights of 16 keys add up to more than this
constexpr int kMostSplits = 4;          // (clusters of eight blocks of this size do not all run at once)
constexpr float kLog2eF = 1.4426950408889634f;

struct PromptParams {
  void* out;
  int out_row_stride;
  const float4* runs;       // [rows][kv_heads][blocks * page_size / 16]
  const int* query_start_loc;
  const int* context_lens;
  const int* seq_index;
  int all_runs;             // in all of `runs`, which has room for kRuns more
  int heads, kv_heads, page_size, blocks;
  int window, keep_first;
  float cap;                // capped scores: cap * log2(e), the pages' f being scale / cap; else 0
  int* error_flag;
  const float* sink;
  const float* q_factors;   // of queries in two halves [tokens][heads]
  int tokens;
  int splits;               // blocks, a cluster, that share a tile's keys
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tanh_fast(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.885390082f));
  return 1.f - __fdividef(2.f, 1.f + e);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void tmem_load16(unsigned taddr, unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_store16(unsigned taddr, const unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// The loads so far are there.  (The registers pass through, so that nothing is done with them before.)
__device__ __forceinline__ void tmem_arrived(unsigned (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :: "memory");
}
// A word with its `n` lowest bits set.
__device__ __forceinline__ unsigned lowest(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
// The 64 threads of two warps meet, and learn whether one of them brings true.
__device__ __forceinline__ bool either(int barrier, bool mine) {
  unsigned r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(barrier), "r"((unsigned)mine) : "memory");
  return r != 0;
}
__device__ __forceinline__ void meet(int barrier) { asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory"); }
__device__ __forceinline__ void tma_load_3d(unsigned dst, const CUtensorMap* map, unsigned bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar) : "memory");
}

// X tiles of 128 rows a block, each with eight softmax warps, scores and accumulator of its own; they share the loader, the issuing
// warp and the ring of keys and values.  Its slots hold 128 keys or 128 values, in turn: tile t's are the numbers 2t and 2t + 1.
// (Q, pieces x X tiles of it, and the slots are what shared memory holds.)
template <int D, int Q> struct PromptSlots { static constexpr int value = D == 64 ? 8 : Q == 1 ? 6 : 5; };
// Tile t's scales come with its keys, into one of these in turn: before tile t's keys are asked for, a slot of tile t - 3's values or of tile
// t - 4's keys (with 8 slots) is free, so that tile t - 4's (t - 5's) softmax is through with its.
template <int D> struct PromptScales { static constexpr int value = D == 64 ? 8 : 4; };
// Warp 0 loads, warp 1 issues, from warp 4 on the softmax, eight warps a tile: two threads a row, of a tile's 64 lower and 64 upper keys.
template <int X> constexpr int prompt_threads() { return 128 + 256 * X; }

// What a run's scales make of a score, y = f s + d, and of a weight for the denominator, z; v: 2^d.  Scores that are not seen (`seen`: a bit a key)
// go out of the way, and with capped scores the others are capped.
struct Terms { float f, d, z, v; };
template <bool kCapped>
__device__ __forceinline__ Terms enter_run(unsigned (&v)[16], const float4 c, bool change, unsigned seen, float cap) {
  if (!change) return Terms{c.x, c.y, c.z, c.w};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (kCapped) v[j] = __float_as_uint(cap * tanh_fast(__uint_as_float(v[j]) * c.x));
    v[j] = (seen >> j) & 1 ? v[j] : 0xff800000u;
  }
  // (a run that the row does not see has no page, and what stands there may be anything)
  const bool none = (seen & 0xffffu) == 0;
  return Terms{kCapped || none ? 1.f : c.x == 0.f ? 1e-37f : c.x, none ? 0.f : c.y, none ? 0.f : c.z, none ? 1.f : c.w};
}

// A row's reference taken anew from the scores of a tile, by its two threads, and its accumulator (each thread's half) brought in line.
// Returns the reference and the factor of what was summed so far.
struct Settle {
  unsigned columns, accumulator;      // of the thread's scores and half of the accumulator
  const float4* run;
  float* between;
  float cap, r, q_factor;
  unsigned seen0, seen1;
  int pair;
  bool upper, rescale;
};
template <int D, bool kCapped>
__device__ __noinline__ float2 settle_rows(const Settle a) {
  unsigned v[16];
  float mx = -INFINITY;
#pragma unroll 1
  for (int g = 0; g < 4; ++g) {
    tmem_load16(a.columns + g * 16, v);
    tmem_arrived(v);
    float4 c = a.run[g];
    c.x *= a.q_factor;
    const Terms e = enter_run<kCapped>(v, c, true, (g < 2 ? a.seen0 : a.seen1) >> (g % 2 * 16), a.cap);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; j += 2) top = max3(top, __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
    mx = fmaxf(mx, fmaf(top, e.f, e.d));
  }
  if (a.upper) *a.between = mx;
  meet(a.pair);
  if (!a.upper) *a.between = mx = fmaxf(mx, *a.between);
  meet(a.pair);
  mx = *a.between;
  float r = a.r, alpha = 1.f;
  if (mx - r > kHeadroom) {       // also when r is still -inf and a score is not
    r = floorf(mx - kHeadroom);       // (a whole number, which nothing is rounded for where it is subtracted)
    alpha = ex2(a.r - r);
  }
  if (a.rescale) {
#pragma unroll 1
    for (int part = 0; part < D / 32; ++part) {
      tmem_load16(a.accumulator + part * 16, v);
      tmem_arrived(v);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
      tmem_store16(a.accumulator + part * 16, v);
    }
    tmem_store_wait();
    tcgen05_fence_before();
  }
  return make_float2(r, alpha);
}

// kTwo: queries and results of 32 bits (one tile a block).  Queries come as two halves each, weights go as two: of both, 22 bits.
// kSplit: the blocks of a cluster share the keys of one tile of queries, a run of steps each, and add their results up through distributed
// shared memory: for launches of few blocks, which take as long as a chain of steps does.
template <int D, int X, bool kCapped, bool kTwo, bool kSplit>
__global__ void __launch_bounds__(prompt_threads<X>(), 1)
attention_int8_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
  extern __shared__ unsigned char smem_raw[];
  const unsigned base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  constexpr int kSub = D / 64;                                      // sub-tiles of 64 dimensions
  constexpr unsigned kKeySubBytes = kKeys * 64 * 2, kRowSubBytes = kRows * 64 * 2, kSlotBytes = kSub * kKeySubBytes;
  static_assert(X == 1 || (!kTwo && !kSplit), "a block's shared and tensor memory");
  constexpr int kPieces = kTwo ? 2 : 1, kSlots = PromptSlots<D, X * kPieces>::value, kScaleSlots = PromptScales<D>::value;
  const unsigned q_smem = base, ring = q_smem + X * kPieces * kSub * kRowSubBytes, scales = ring + kSlots * kSlotBytes;
  const unsigned bars = scales + kScaleSlots * kRuns * 16;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kSlots + s); };
  const unsigned q_full = bars + 8u * (2 * kSlots);
  auto tile_bar = [&](int x, int which) { return q_full + 8u * (1 + x * 3 + which); };
  const unsigned drained = tile_bar(X, 0);
  __shared__ unsigned tmem_slot;
  __shared__ float between[X][kRows];       // a row's two threads
  unsigned char* generic_base = smem_raw + (base - smem_addr(smem_raw));
  float* const held = reinterpret_cast<float*>(generic_base + (ring - base));       // [D + 2][rows], where the ring was: sums, references, their sums

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();       // (by now all that came before the pages were spread is done)
  const int seq = p.seq_index ? p.seq_index[blockIdx.y] : blockIdx.y;
  if (seq < 0) return;        // a place of padding in the list of sequences
  const int splits = kSplit ? p.splits : 1, split = (int)blockIdx.x % splits, kvh = (int)blockIdx.x / splits;
  const int q_begin = p.query_start_loc[seq], q_len = p.query_start_loc[seq + 1] - q_begin;
  const int groups = p.heads / p.kv_heads, tq = kRows / groups;
  // The last query tiles see the most keys: they are handed out first.
  const int block_q0 = (int)(gridDim.z - 1 - blockIdx.z) * X * tq;
  if (block_q0 >= q_len) return;
  const int ctx = p.context_lens[seq];
  const int block_q = min(X * tq, q_len - block_q0);
  const int hi = ctx - q_len + block_q0 + block_q, lo = first_visible(ctx - q_len + block_q0, p.window);
  // The warp's own tile: its queries and positions.
  const int x = X == 1 || warp < 4 ? 0 : (warp - 4) >> 3;
  const int q0 = block_q0 + x * tq, tile_q = max(0, min(tq, q_len - q0)), rows_used = tile_q * groups;
  const int first_qpos = ctx - q_len + q0, last_qpos = first_qpos + max(tile_q, 1) - 1;
  const unsigned s_full = tile_bar(x, 0), p_full = tile_bar(x, 1), pv_done = tile_bar(x, 2);
  const int tile_lo = lo / kKeys, tile_hi = (hi + kKeys - 1) / kKeys;
  const int kept_end = p.keep_first > 0 ? min(p.keep_first, lo) : 0;       // first keys that stay visible behind the window
  const int kept_tiles = min((kept_end + kKeys - 1) / kKeys, tile_lo);
  const int all_tiles = kept_tiles + tile_hi - tile_lo, first_tile = all_tiles * split / splits;
  const int ntiles = all_tiles * (split + 1) / splits - first_tile;       // of this block
  auto tile_at = [&](int t) { return t + first_tile < kept_tiles ? t + first_tile : tile_lo + t + first_tile - kept_tiles; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(drained, 1);
    for (int t = 0; t < X; ++t) {
      mbar_init(tile_bar(t, 0), 1);
      mbar_init(tile_bar(t, 1), 8);
      mbar_init(tile_bar(t, 2), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  constexpr unsigned kTmemCols = X * (128 + D) + (kTwo ? D : 0) <= 256 ? 256u : 512u;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Warp 0 asks for a slot's 128 keys or values (with both's scales), a box for every 64 dimensions.  (What lies behind the context is the
  // next head's, or zeros behind the last, and masked either way; the scales have room for a tile behind the last.)
  const int first_row = ((int)blockIdx.y * p.kv_heads + kvh) * p.blocks * p.page_size;
  auto load_slot = [&](int i, bool slot_is_new) -> bool {
    const int slot = i % kSlots, t = i >> 1, row = first_row + tile_at(t) * kKeys;
    if (!slot_is_new && !warp_wait(empty(slot), ((unsigned)(i / kSlots) & 1) ^ 1, p.error_flag, 51)) return false;
    if (elected()) {
      mbar_expect_tx(full(slot), kSlotBytes + ((i & 1) ? 0 : kRuns * 16));
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub)
        tma_load_2d(ring + slot * kSlotBytes + sub * kKeySubBytes, (i & 1) ? &map_v : &map_k, full(slot), sub * 64, row);
      if (!(i & 1)) bulk_load(scales + (t % kScaleSlots) * (kRuns * 16), p.runs + min(row / 16, p.all_runs), kRuns * 16, full(slot));
    }
    return true;
  };
  const int ahead = min(kSlots, 2 * ntiles);
  if (warp == 0) {
    // A tile of queries: the heads of a group, a query behind the other, are its rows.  (Those behind the portion are masked; those that the
    // box does not reach, of groups that do not divide 128, are never written: whatever stands there stays in its row.)
    if (elected()) {
      mbar_expect_tx(q_full, X * kPieces * D * 2 * tq * groups);
#pragma unroll
      for (int i = 0; i < X * kPieces * kSub; ++i)
        tma_load_3d(q_smem + i * kRowSubBytes, &map_q, q_full, i % kSub * 64, kvh * groups, q_begin + block_q0 + i / kSub * (kTwo ? p.tokens : tq));
    }
    for (int i = 0; i < ahead; ++i) load_slot(i, true);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const unsigned tmem_base = tmem_slot;
  const unsigned tmem_s = tmem_base + x * 128u, tmem_o = tmem_base + X * 128u + x * D, tmem_second = tmem_o + D;

  if (warp == 0) {
    // ------------------------------------------------------------------ loader
    int asked = ahead;
    while (asked < 2 * ntiles && load_slot(asked, false)) ++asked;
    // Nobody leaves before what was asked for has come, also where there was nothing to do with it or a wait gave up.
    warp_wait(q_full, 0, p.error_flag, 54);
    for (int i = max(0, asked - kSlots); i < asked; ++i) warp_wait(full(i % kSlots), (unsigned)(i / kSlots) & 1, nullptr, 0);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer
    {
      // 32-bit sums, M 128.  S: bfloat16 (halves), N 128.  P V: halves, N = D, the second operand N-major, its sub-tiles of 64 dimensions
      // kKeySubBytes apart (the descriptor's leading offset).
      constexpr unsigned idesc_qk = (1u << 4) | (kTwo ? 0u : (1u << 7) | (1u << 10)) | ((unsigned)(kKeys >> 3) << 17) | ((unsigned)(kRows >> 4) << 24);
      constexpr unsigned idesc_pv = (1u << 4) | (1u << 16) | ((unsigned)(D >> 3) << 17) | ((unsigned)(kRows >> 4) << 24);
      const unsigned long long desc_q = umma_desc(q_smem), desc_k = umma_desc(ring);
      unsigned long long desc_v = desc_k;
      if (kSub > 1) desc_v = (desc_v & ~(0x3fffULL << 16)) | ((unsigned long long)((kKeySubBytes >> 4) & 0x3fff) << 16);
      // The weights of tile t - 1 lie where S of tile t goes: the tensor cores are through with them first, they take one product after
      // another.  So do the query tiles: the second's products come behind all of the first's, and from then on one's softmax runs
      // while the other's products do.
      auto arrived = [&](int i) { return warp_wait(full(i % kSlots), (unsigned)(i / kSlots) & 1, p.error_flag, 53); };
      auto issue_qk = [&](int t, int tile) {
        const int slot = (2 * t) % kSlots;
        const unsigned long long dq = desc_q + (unsigned long long)((tile * kSub * kRowSubBytes) >> 4);
        const unsigned long long dk = desc_k + (unsigned long long)((slot * kSlotBytes) >> 4);
        if (elected()) {
#pragma unroll
          for (int i = 0; i < kPieces * D / 16; ++i) {
            const int k = i % (D / 16), piece = kPieces - 1 - i / (D / 16);       // (the small one first: less is cut off)
            umma_bf16(tmem_base + tile * 128u, dq + (unsigned long long)(((piece * kSub + k / 4) * kRowSubBytes + (k % 4) * 32) >> 4),
                      dk + (unsigned long long)(((k / 4) * kKeySubBytes + (k % 4) * 32) >> 4), idesc_qk, i > 0);
          }
          umma_commit(tile_bar(tile, 0));
          if (tile == X - 1) umma_commit(empty(slot));
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int tile) -> bool {
        const int slot = (2 * t + 1) % kSlots;
        const unsigned long long dv = desc_v + (unsigned long long)((slot * kSlotBytes) >> 4);
        if (!warp_wait(tile_bar(tile, 1), (unsigned)t & 1, p.error_flag, 55)) return false;
        tcgen05_fence_after();
        if (elected()) {
#pragma unroll
          for (int i = 0; i < kPieces * kKeys / 16; ++i)       // (the instruction is the one of bfloat16: the types are the descriptor's)
            umma_bf16_ts(tmem_base + X * 128u + tile * D, tmem_base + tile * 128u + (i + (kPieces - 1) * (kKeys / 16)) % (kPieces * kKeys / 16) * 8u,
                         dv + (unsigned long long)((i % (kKeys / 16) * 16 * 128) >> 4), idesc_pv, (!kTwo && t > 0) || i > 0);
          if (tile == X - 1) umma_commit(empty(slot));
          if (t + 1 == ntiles) umma_commit(tile_bar(tile, 2));
        }
        __syncwarp();
        return true;
      };
      bool ok = ntiles > 0 && warp_wait(q_full, 0, p.error_flag, 54) && arrived(0);
      if (ok) tcgen05_fence_after();
      for (int tile = 0; ok && tile < X; ++tile) issue_qk(0, tile);
      for (int t = 0; ok && t < ntiles; ++t) {
        ok = arrived(2 * t + 1) && (t + 1 == ntiles || arrived(2 * t + 2));       // (nothing to wait for between P and the next S)
        for (int tile = 0; ok && tile < X; ++tile) {
          ok = issue_pv(t, tile);
          if (ok && t + 1 < ntiles) issue_qk(t + 1, tile);
        }
      }
      if (!ok && ntiles > 0) {        // products that are under way still are done before tensor memory goes back
        if (elected()) umma_commit(drained);
        warp_wait(drained, 0, nullptr, 0);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const bool upper = ((warp - 4) >> 2) & 1;
    const unsigned lane_field = (unsigned)(quarter * 32) << 16;
    const int qpos = row < rows_used ? first_qpos + row / groups : -1;
    const int row_lo = first_visible(qpos, p.window), last_lo = first_visible(last_qpos, p.window);
    const unsigned columns = tmem_s + lane_field + upper * 64;
    const int pair = 1 + x * 4 + quarter;       // the barrier of a row's two threads' warps
    const float q_factor = kTwo && row < rows_used ? p.q_factors[(size_t)(q_begin + q0 + row / groups) * p.heads + kvh * groups + row % groups] : 1.f;
    float r = -INFINITY, l = 0.f;
    // (A wait that ran out lets the rest run to its end: the two warps of a pair meet in every tile.)
    bool ok = ntiles > 0;
    for (int t = 0; t < ntiles; ++t) {
      const int key0 = tile_at(t) * kKeys + upper * 64;
      const bool all_seen = key0 + 63 <= first_qpos && key0 >= last_lo && qpos >= 0;
      // S is there, and P V of the tile before is done with the accumulator: it came first.
      ok = ok && mbar_wait(s_full, (unsigned)t & 1, p.error_flag, 56);
      tcgen05_fence_after();
      __syncwarp();
      unsigned s[2][16];
      tmem_load16(columns, s[0]);
      // What the scales make of run g of 16 keys: of a score y = f s + d, of a weight for the denominator z.  (They came with the keys, and S
      // was made after that.)
      const float4* run = reinterpret_cast<const float4*>(generic_base + (scales - base)) + (t % kScaleSlots) * kRuns + upper * 4;
      unsigned seen[2] = {~0u, ~0u};         // the row's keys
      if (!all_seen) {
#pragma unroll
        for (int c = 0; c < 2; ++c) seen[c] = lowest(qpos + 1 - key0 - 32 * c) & (~lowest(row_lo - key0 - 32 * c) | lowest(p.keep_first - key0 - 32 * c));
      }
      // Value rows of keys outside [lo, hi) may hold anything: zero them before P V reads them.
      if (key0 < lo || key0 + 64 > hi) {
        const int i = 2 * t + 1, slot = i % kSlots;
        ok = ok && mbar_wait(full(slot), (unsigned)(i / kSlots) & 1, p.error_flag, 57);
        unsigned char* vt = generic_base + (ring - base) + slot * kSlotBytes;
        for (int e = (warp & 3) * 32 + lane; e < kSub * 64 * 8; e += 128) {
          const int sub = e / (64 * 8), key = (e >> 3) % 64, kpos = key0 + key;
          if ((kpos < lo && kpos >= kept_end) || kpos >= hi)
            *reinterpret_cast<uint4*>(vt + sub * kKeySubBytes + (upper * 64 + key) * 128 + ((e & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();
        __syncwarp();
      }
      // Of 32 bits, what the step before gave is added to a second accumulator here: the tensor cores cut off what they add rather than round it,
      // which adds up (2,100 keys, 32 heads on 8 of 128: 5.4e-6 of the result without, 4.7e-7 with, 1.1e-6 a form in 32 bits throughout).
      if (kTwo && t > 0) {
        unsigned o[16], more[16];
#pragma unroll 1
        for (int part = 0; part < D / 32; ++part) {
          tmem_load16(tmem_o + lane_field + upper * (D / 2) + part * 16, o);
          tmem_load16(tmem_second + lane_field + upper * (D / 2) + part * 16, more);
          tmem_load_wait();
          if (t > 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(more[j]));
          }
          tmem_store16(tmem_second + lane_field + upper * (D / 2) + part * 16, o);
        }
        tmem_store_wait();
      }
      unsigned packed[kPieces][32];
      float sum;
      // A row's reference r moves only when the weights grow out of a half's range, and that is found then: the sums tell.  (So no score is
      // compared in passing.)  Both warps of the rows meet for it, and go back to the scores; in the first tile they begin so.
      bool settled = t == 0;
      auto settle = [&] {
        const float2 now = settle_rows<D, kCapped>(Settle{columns, (kTwo ? tmem_second : tmem_o) + lane_field + upper * (D / 2), run, &between[x][row], p.cap, r, q_factor, seen[0], seen[1], pair,
                                                          upper, t > 0});
        r = now.x;
        l *= now.y;
      };
      if (settled) settle();
#pragma unroll 1
      for (;;) {
        float most = 0.f;
        sum = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          unsigned(&v)[16] = s[g & 1];
          tmem_arrived(v);
          if (g < 3) tmem_load16(columns + (g + 1) * 16, s[(g + 1) & 1]);
          float4 c = run[g];
          if constexpr (kTwo) c.x *= q_factor;
          const Terms e = enter_run<kCapped>(v, c, kCapped || !all_seen, seen[g / 2] >> (g % 2 * 16), p.cap);
          // (Of 32 bits, 2^d comes as a factor behind the exponential: the sum of d and r would be rounded.)
          const float d = kTwo && e.d != -INFINITY ? 0.f : e.d;
          const float2 factor = both(e.f), shift = both(r == -INFINITY ? d : d - r);
          float2 part = both(0.f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 y = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), factor, shift);
            float2 w = make_float2(ex2(y.x), ex2(y.y));
            part = add2(part, w);
            if constexpr (kTwo) w = mul2(w, both(e.v));
            packed[0][g * 8 + i] = pack_half(w.x, w.y);
            if constexpr (kTwo) {
              const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&packed[0][g * 8 + i]));
              packed[kPieces - 1][g * 8 + i] = pack_half(w.x - back.x, w.y - back.y);
            }
          }
          most = fmaxf(most, kTwo ? (part.x + part.y) * e.v : part.x + part.y);
          sum = fmaf(part.x + part.y, kTwo ? 1.f : e.z, sum);
        }
        if (settled) {
          meet(pair);       // both halves of the accumulator are rescaled, and the scores read
          break;
        }
        if (!either(pair, most > kLargest || (r == -INFINITY && qpos >= 0))) break;
        settle();
        settled = true;
        tmem_load16(columns, s[0]);
      }
      l += sum;
      // The weights go over the lower half's scores, what they leave over the upper half's.
      tmem_store32(tmem_s + lane_field + upper * 32, packed[0]);
      if constexpr (kTwo) tmem_store32(tmem_s + lane_field + 64 + upper * 32, packed[1]);
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    // Output: wait for the last P V, read a row (each thread half of it), divide by the row's sum, store.
    ok = ok && mbar_wait(pv_done, 0, p.error_flag, 59);
    if (upper) between[x][row] = l;
    meet(pair);
    if (!upper) between[x][row] = l += between[x][row];
    meet(pair);
    l = between[x][row];
    if (!kSplit && p.sink != nullptr && row < rows_used) l += exp2f(p.sink[kvh * groups + row % groups] * kLog2eF - r);
    if (kSplit) {
      // Sums that are not divided yet, a column behind the other.
      if (ok) {
        tcgen05_fence_after();
#pragma unroll 1
        for (int part = 0; part < D / 32; ++part) {
          unsigned o[16];
          __syncwarp();
          tmem_load16(tmem_o + lane_field + upper * (D / 2) + part * 16, o);
          tmem_load_wait();
          if (kTwo && ntiles > 1) {
            unsigned more[16];
            tmem_load16(tmem_second + lane_field + upper * (D / 2) + part * 16, more);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(more[j]));
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) held[(upper * (D / 2) + part * 16 + j) * kRows + row] = __uint_as_float(o[j]);
        }
      }
      if (!upper) {
        held[D * kRows + row] = ok ? r : -INFINITY;
        held[(D + 1) * kRows + row] = l;
      }
    } else if (ok) {
      tcgen05_fence_after();
      const int qi = q0 + row / groups, head = kvh * groups + row % groups;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const size_t place = (size_t)(q_begin + qi) * p.out_row_stride + (size_t)head * D + upper * (D / 2);
      unsigned o[D / 64][32];
      __syncwarp();
#pragma unroll
      for (int part = 0; part < D / 64; ++part) tmem_load32(tmem_o + lane_field + upper * (D / 2) + part * 32, o[part]);
      tmem_load_wait();
      if (kTwo && ntiles > 1) {
#pragma unroll
        for (int part = 0; part < D / 32; ++part) {
          unsigned more[16];
          tmem_load16(tmem_second + lane_field + upper * (D / 2) + part * 16, more);
          tmem_load_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) o[part / 2][part % 2 * 16 + j] = __float_as_uint(__uint_as_float(o[part / 2][part % 2 * 16 + j]) + __uint_as_float(more[j]));
        }
      }
      if (row < rows_used) {
        if constexpr (kTwo) {
          float* dst = (float*)p.out + place;
#pragma unroll
          for (int v = 0; v < D / 8; ++v) {
            const unsigned* from = &o[v / 8][v % 8 * 4];
            *reinterpret_cast<float4*>(dst + v * 4) = make_float4(__uint_as_float(from[0]) * inv, __uint_as_float(from[1]) * inv,
                                                                  __uint_as_float(from[2]) * inv, __uint_as_float(from[3]) * inv);
          }
        } else {
          bf16* dst = (bf16*)p.out + place;
#pragma unroll
          for (int v = 0; v < D / 16; ++v) {
            unsigned w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const unsigned* from = &o[v / 4][v % 4 * 8 + 2 * e];
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(from[0]) * inv, __uint_as_float(from[1]) * inv);
              w[e] = *reinterpret_cast<const unsigned*>(&h);
            }
            *reinterpret_cast<uint4*>(dst + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tcgen05_fence_before();
  if constexpr (kSplit) {
    cluster_sync_all();       // every block's sums are in place (release / acquire)
    if (warp >= 4) {
      // A row is two threads', each with half of this block's share of the columns.
      const int row = threadIdx.x & (kRows - 1), columns = D / splits / 2, c0 = split * (D / splits) + ((int)threadIdx.x - 128) / kRows * columns;
      auto remote = [&](int at, int rank) {
        unsigned addr;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(held + at)), "r"(rank));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
        return v;
      };
      if (row < rows_used) {
        float w[kMostSplits], top = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < kMostSplits; ++i) {
          w[i] = i < splits ? remote(D * kRows + row, i) : -INFINITY;
          top = fmaxf(top, w[i]);
        }
#pragma unroll
        for (int i = 0; i < kMostSplits; ++i) {
          // A block that saw no key brings neither a reference nor a sum.  One whose scores are all NaN brings no reference either (a maximum
          // passes NaN over), but its sum is NaN, and so is the row.
          const float sum = i < splits ? remote((D + 1) * kRows + row, i) : 0.f;
          w[i] = w[i] != -INFINITY ? exp2f(w[i] - top) : sum == 0.f ? 0.f : NAN;
          if (w[i] != 0.f) l += w[i] * sum;
        }
        const int qi = q0 + row / groups, head = kvh * groups + row % groups;
        if (p.sink != nullptr) l += exp2f(p.sink[head] * kLog2eF - top);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t place = (size_t)(q_begin + qi) * p.out_row_stride + (size_t)head * D;
        for (int c = c0; c < c0 + columns; c += 4) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kMostSplits; ++i)
            if (w[i] != 0.f) {      // (a NaN is not)
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[j] = fmaf(w[i], remote((c + j) * kRows + row, i), sum[j]);
            }
          if constexpr (kTwo) {
            *reinterpret_cast<float4*>((float*)p.out + place + c) = make_float4(sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
          } else {
            const __nv_bfloat162 a = __floats2bfloat162_rn(sum[0] * inv, sum[1] * inv), b = __floats2bfloat162_rn(sum[2] * inv, sum[3] * inv);
            *reinterpret_cast<uint2*>((bf16*)p.out + place + c) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
          }
        }
      }
    }
    cluster_sync_all();       // nobody leaves while another reads
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// Queries [tokens, heads, head_dim], boxes of tq queries x the heads of a group x 64 dimensions.
static bool query_map(CUtensorMap* map, const void* q, long long row_stride, long long tokens, int heads, int head_dim, int groups, int tq, bool halves) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)groups, (cuuint32_t)tq};
  const cuuint32_t elem[3] = {1, 1, 1};
  return encode(map, halves ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of `head_dim` 16-bit numbers, boxes of 128 rows x 64 dimensions.
static bool tile_map(CUtensorMap* map, const void* ptr, long rows, int head_dim, bool halves) {
  EncodeTiledFn encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)head_dim * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)kKeys};
  const cuuint32_t elem[2] = {1, 1};
  return encode(map, halves ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides,
                box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int X, bool kCapped, bool kTwo, bool kSplit>
static int launch_prompt_as(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PromptParams& p, dim3 grid, cudaStream_t stream) {
  constexpr int kTiles = kTwo ? 2 : X, kSlots = PromptSlots<D, kTiles>::value, kScaleSlots = PromptScales<D>::value;
  constexpr size_t smem = (size_t)kTiles * kRows * D * 2 + kSlots * (size_t)kKeys * D * 2 + kScaleSlots * kRuns * 16 + 8 * (2 * kSlots + 2 + 3 * X) + 1024;
  static_assert(smem + X * 4 * kRows + 16 <= 232448, "more shared memory than a block may have");
  static_assert(!kSplit || (D + 2) * kRows * 4 <= kSlots * kKeys * D * 2, "sums where the ring was");
  auto kernel = attention_int8_prompt_kernel<D, X, kCapped, kTwo, kSplit>;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  if constexpr (!kSplit) return (int)launch_pdl(0, kernel, grid, dim3(prompt_threads<X>()), smem, stream, mq, mk, mv, p);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid.x * p.splits, grid.y, grid.z);
  config.blockDim = dim3(prompt_threads<X>());
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = p.splits;
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = pdl_enabled(0) ? 2 : 1;
  return (int)cudaLaunchKernelEx(&config, kernel, mq, mk, mv, p);
}
template <int D, int X, bool kTwo = false>
static int launch_prompt(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PromptParams& p, dim3 grid, cudaStream_t stream) {
  if constexpr (X == 1)
    if (p.splits > 1)
      return p.cap > 0.f ? launch_prompt_as<D, X, true, kTwo, true>(mq, mk, mv, p, grid, stream)
                         : launch_prompt_as<D, X, false, kTwo, true>(mq, mk, mv, p, grid, stream);
  return p.cap > 0.f ? launch_prompt_as<D, X, true, kTwo, false>(mq, mk, mv, p, grid, stream)
                     : launch_prompt_as<D, X, false, kTwo, false>(mq, mk, mv, p, grid, stream);
}

}  // namespace li

using namespace li;

LI_EXPORT int li_attention_int8_prompt_supports(int heads, int kv_heads, int head_dim, int page_size) {
  if (kv_heads < 1 || kv_heads > 256 || heads < 1 || heads % kv_heads || heads / kv_heads > kRows) return 0;
  return (head_dim == 64 || head_dim == 128) && page_size >= 16 && page_size % 16 == 0;
}

struct AttentionInt8PromptArgs {
  long long dtype;          // of q and out
  const void* q;            // [tokens, heads, head_dim]
  long long tokens;
  long long q_row_stride;
  void* out;
  long long out_row_stride;
  const void *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int* block_table;
  long long table_stride;
  const int *query_start_loc, *context_lens, *seq_index;
  long long num_seqs, max_q_len, heads, kv_heads, head_dim, page_size, num_pages;
  double scale;
  long long window, keep_first;
  double softcap;
  const float* sink;
  void* work;               // 16-byte aligned: keys and values of num_seqs * blocks pages in 16 bits, 16 bytes for 16 of them and 128 more;
                            // for float32, 4 head_dim + 4 bytes for each of tokens x heads behind that
  long long blocks;         // of a sequence, at most: every context fits them
  int* error_flag;          // device int, zero: the number (51 to 60) of a bounded wait that gave up
  cudaStream_t stream;
};

LI_EXPORT int li_attention_int8_prompt(const AttentionInt8PromptArgs* a) {
  const int rows = (int)a->num_seqs, kv_heads = (int)a->kv_heads, page_size = (int)a->page_size, D = (int)a->head_dim, blocks = (int)a->blocks;
  if (rows == 0 || a->max_q_len == 0 || blocks == 0) return 0;
  if (!li_attention_int8_prompt_supports((int)a->heads, kv_heads, D, page_size) || rows > 65535) return LI_ERR_UNSUPPORTED;
  if ((long)rows * kv_heads * blocks * page_size > 0x7fffffffL) return LI_ERR_UNSUPPORTED;
  const bool two_pieces = a->dtype == kFloat32;
  const int per16 = two_pieces ? 4 : 8;
  if (!aligned16(a->q) || a->q_row_stride % per16 || !aligned16(a->out) || a->out_row_stride % per16 || !aligned16(a->k_pool) ||
      !aligned16(a->v_pool) || !aligned16(a->work))
    return LI_ERR_ALIGNMENT;
  if (a->tokens * a->heads > 0x3fffffffL) return LI_ERR_UNSUPPORTED;
  const size_t bytes = (size_t)rows * blocks * kv_heads * page_size * D * 2;
  unsigned char* const work = (unsigned char*)a->work;
  const bool capped = a->softcap > 0;
  const int keep_first = a->window > 0 ? (int)a->keep_first : 0;
  ExpandParams e{{(const signed char*)a->k_pool, (const signed char*)a->v_pool}, {a->k_scale, a->v_scale}, a->block_table,
                 (int)a->table_stride, a->query_start_loc, a->context_lens, a->seq_index, (int)a->window, keep_first,
                 fabsf(capped ? (float)(a->scale / a->softcap) : (float)a->scale * kLog2eF), a->scale < 0 ? 0x80008000u : 0u, {(uint4*)work, (uint4*)(work + bytes)},
                 (float4*)(work + 2 * bytes), blocks, kv_heads, D, page_size, (int)a->num_pages, two_pieces};
  long long parts = 1;      // a page is a block's, and of several while they are not many a multiprocessor (1,024 queries behind 3,000, 32 heads on 8
                            // of 128: the call takes 84 us with a block a page, 80 with four)
  while (parts < 4 && parts * 2 * 256 <= (long long)kv_heads * page_size * D / 16 && parts * blocks * rows <= 4 * 148) parts *= 2;
  const long all = (long)rows * kv_heads * blocks * page_size;
  __half* const pieces = (__half*)(work + 2 * bytes + all + 128);
  float* const factors = (float*)(pieces + 2 * (size_t)a->tokens * a->heads * D);
  if (two_pieces) {
    const cudaError_t split = launch_pdl(rows, split_queries_kernel, dim3((unsigned)((a->tokens * a->heads + 7) / 8)), dim3(256), 0, a->stream, (const float*)a->q,
                                         (int)a->q_row_stride, pieces, factors, (int)a->tokens, (int)a->heads, D);
    if (split != cudaSuccess) return (int)split;
  }
  const cudaError_t status = launch_pdl(rows, expand_pages_int8_kernel, dim3(blocks, 2 * (unsigned)parts, rows), dim3(256), 0, a->stream, e);
  if (status != cudaSuccess) return (int)status;
  static const int sms = [] {
    int device = 0, n = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) n = 148;
    return n;
  }();
  const int groups = (int)(a->heads / kv_heads), tq = kRows / groups;
  CUtensorMap mq, mk, mv;
  if (!(two_pieces ? query_map(&mq, pieces, a->heads * D, 2 * a->tokens, (int)a->heads, D, groups, tq, true)
                   : query_map(&mq, a->q, a->q_row_stride, a->tokens, (int)a->heads, D, groups, tq, false)) ||
      !tile_map(&mk, work, all, D, two_pieces) || !tile_map(&mv, work + bytes, all, D, true))
    return LI_ERR_UNSUPPORTED;
  PromptParams p{a->out, (int)a->out_row_stride, e.runs, a->query_start_loc, a->context_lens,
                 a->seq_index, (int)(all / 16), (int)a->heads, kv_heads, page_size, blocks, (int)a->window, keep_first,
                 capped ? (float)a->softcap * kLog2eF : 0.f, a->error_flag, a->sink, factors, (int)a->tokens, 1};
  // How many steps of 128 keys a block takes, at most and (its portion's first tile, where no window evens them out) at least.
  long most_keys = (long)blocks * page_size, least_keys = most_keys - a->max_q_len;
  if (a->window > 0 && a->window + tq + keep_first < most_keys) most_keys = least_keys = a->window + tq + keep_first;
  const double most = (double)most_keys / kKeys, least = (double)(least_keys < 0 ? 0 : least_keys) / kKeys;
  const long single_tiles = (a->max_q_len + tq - 1) / tq, singles = single_tiles * rows * kv_heads;
  // Two tiles of queries a block: a step takes 3,500 cycles then, and some 2,800 with one tile.  One where such blocks all have an SM of their own,
  // or where the second round's, short ones behind long ones of the first, leave it the shorter of the two (3,000 tokens behind 500, 8 heads
  // of 64: 56 us of one tile, 75 of two; 1,024 behind 3,000, 32 heads on 8 of 128: 109 and 85).
  bool two = singles > sms && !two_pieces;
  if (two && singles <= 2 * sms) {
    const double both_rounds = 2 * most - (most - least) * 2 * sms / singles;
    two = 2800 * (both_rounds > most ? both_rounds : most) >= 3500 * most;
  }
  const long tiles = two ? (a->max_q_len + 2 * tq - 1) / (2 * tq) : single_tiles;
  if (tiles > 65535) return LI_ERR_UNSUPPORTED;
  const dim3 grid(kv_heads, rows, (unsigned)tiles);
  if (!two) {
    // Blocks share a tile's keys while all of them run at once, three steps each at least (5 portions of 8 tokens behind 4,339, 28 heads on
    // 4 of 128: 74 us unshared, 33 by fours); and by twos where that makes up for the four steps or so that sharing costs because the short
    // tiles' fill the SMs behind the long ones' (3,536 tokens in 2 portions behind 1,131, 2 heads of 64: 44 us, 29 by twos).
    while (p.splits < kMostSplits && 2 * p.splits * singles <= sms && most >= 6 * p.splits) p.splits *= 2;
    if (p.splits == 1 && singles <= sms && most >= 6 && (most - least) * sms / (2 * singles) > 4) p.splits = 2;
  }
  if (two_pieces) return D == 64 ? launch_prompt<64, 1, true>(mq, mk, mv, p, grid, a->stream) : launch_prompt<128, 1, true>(mq, mk, mv, p, grid, a->stream);
  if (D == 64) return two ? launch_prompt<64, 2>(mq, mk, mv, p, grid, a->stream) : launch_prompt<64, 1>(mq, mk, mv, p, grid, a->stream);
  return two ? launch_prompt<128, 2>(mq, mk, mv, p, grid, a->stream) : launch_prompt<128, 1>(mq, mk, mv, p, grid, a->stream);
}
