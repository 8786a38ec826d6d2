// Paged attention of single decoded tokens over keys and values held in 8 bits (int8_cache.cu); portions of prompts are
// attention_int8_prompt.cu's, and sizes that neither takes read their pages back and go to the kernels of 16 and 32 bits (ops/int8.py).
//
//   out = sum_j w_j s_v(page of j) v_j / sum_j w_j,   w_j = exp(scale * s_k(page of j) * (q . k_j) - max),
//
// k_j, v_j whole numbers, j over the keys that the query sees.  Bound by memory: 2 D bytes a key.
//
// A block owns one (sequence, KV head, split of its keys); each of its four warps walks 16 keys of every 64 and meets the others at
// the end.  A thread asks (cp.async) for the 16 bytes of keys and values that mma.sync wants from it, several groups of 16 keys ahead, into
// places in shared memory that it alone reads: no barrier, no bank conflict, no register waits for memory.  (A trip to memory takes some
// 1,600 cycles here, a group of 16 keys of 64 dimensions 500; with two groups in registers instead, one block an SM took 1,600 a group.)
//
//   S^T = K Q^T   first operand K: thread (g, t) of a warp (g = lane / 4, t = lane % 4) has, of keys g and g + 8, the dimensions
//                 64 c + 16 t ... + 15, and Q is laid out alike (a sum over dimensions does not mind their order).
//   O^T += V^T P^T  first operand V^T: thread (g, t) has, of keys 2t, 2t + 1, 2t + 8, 2t + 9, the dimensions g D/8 ...; byte
//                 permutes pair two keys.  Row i of tile n is dimension g D/8 + 2n (+ 1 for rows 8 up).
//   In between, P^T goes from the layout of a result to that of a second operand by movmatrix.
//
// What sets the pace beside memory is the number of instructions a key costs, so K is not converted at all where Q has 16 bits: each
// head of Q becomes whole numbers of 14 bits and a sign, 128 h + l with h and l of 8 bits, x ~ (128 h + l) max|x| / 16256 (an
// error of 2^-15 of the head's largest number), and m16n8k32 of whole numbers multiplies K with h and with l, exactly.  With Q of 32
// bits, K becomes halves, and Q enters as the sum of two halves, each head divided by a power of two.
// V becomes halves without a conversion: a byte b with its sign bit turned, below the byte 0x64, is the half 1024 + (b + 128), exact; one
// subtraction gives b.
//
// The scale of a page's values cannot go into P as it is (it may have any size, a half may not): the weights that are multiplied
// with values are exp2(s - m) exp2(log2 s_v + m - r) with a running reference r of their own, the ones that are summed for the
// denominator exp2(s - m).  Both references follow the scores only when one outgrows them by 2^7 and 2^16 (r is 2^8 above what keeps the largest
// weight at 1: a half holds 2^15, and weights of 2^-22 of the largest still have all their bits).  All sums are 32-bit; weights are
// rounded to halves, 11 bits (with 32-bit Q to the sum of two).
//
// The splits of a (sequence, KV head) are one thread-block cluster: each leaves its result in its shared memory, and they merge
// through distributed shared memory, a share of the dimensions each.  No partial results in memory, no counters, no atomics.
#include "attention_mma.cuh"
#include "int8.cuh"
#include "tcgen05.cuh"

namespace li {

struct Int8AttnParams {
  const void* q;
  int q_row_stride;
  void* out;
  int out_row_stride;
  const signed char* k_pool;
  const signed char* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int* block_table;
  int table_stride;
  const int* query_start_loc;
  const int* context_lens;
  const int* seq_index;     // optional: batch row of each launched sequence (negative: none)
  int heads, kv_heads, page_size, num_pages;
  float scale;
  int window;               // see first_visible (common.cuh)
  float softcap;            // 0: none
  const float* sink;        // [heads] or null: exp(sink[h]) is one more term of head h's denominator
  bool beside;              // the kernel ahead neither writes what this one reads nor the same results: they run side by side
  bool after_append;        // the kernel ahead is rope_kv_write_int8, and it brings no more than the newest token of these sequences
};

__device__ __forceinline__ uint4 shared16(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 shared8(unsigned addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// Two bytes of a register (the low byte of either half) as two halves.
__device__ __forceinline__ unsigned halves_of(unsigned bytes) {
  unsigned r;
  const unsigned biased = (bytes & 0x00ff00ffu) ^ 0x64806480u;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(biased), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned turned(unsigned m) {      // an 8 x 8 matrix of halves, rows and columns exchanged
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(m));
  return r;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_half(unsigned h) {
  float2 v;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(v.x), "=f"(v.y) : "r"(h));
  return v;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned word4(const uint4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// What the warps, and then the cluster's blocks, leave for the merge: [kWarps][rows][D] sums, maxima and denominators of the warps;
// the block's own result [rows][D] and the base-2 logarithm of its denominator.
template <int D, int kRows> struct Int8Merge {
  float os[kWarps][kRows][D];
  float ms[kWarps][kRows], ls[kWarps][kRows];
  float mine[kRows][D];
  float lse[kRows];
};

// With Q of 16 bits, a warp of head size 64 takes its groups of 16 keys two at a time: two chains of products and exponentials run side by side, and what is
// done once a turn (references, votes, exchanges) is done half as often (128 sequences of 1,000 keys, 8 KV heads: 35.0 us one by one, 32.9
// by twos).  At 128 that takes the registers and the memory of a fourth block an SM (59.5 and 63.3 us).  A warp has room for three
// turns, all but the one it multiplies on their way.
template <typename T, int D> constexpr int kTurn = D == 64 && sizeof(T) == 2 ? 2 : 1;
constexpr int kRing = 3;

constexpr float kQuerySteps = 16256.f;      // 127 * 128: the largest 128 h + l

// T: the type of q and out.  NT: tiles of eight heads.  kCapped: scores are capped.
template <typename T, int D, int NT, bool kCapped>
__device__ __forceinline__ void attend(const Int8AttnParams& p, int splits) {
  constexpr bool kTwo = sizeof(T) == 4;         // Q and P as the sum of two halves
  constexpr int kPieces = kTwo ? 2 : 1;
  constexpr int kRows = NT * 8;
  constexpr int X = kTurn<T, D>;                   // groups a turn
  constexpr unsigned kGroupBytes = 16 * D * 2;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Int8Merge<D, kRows>& merge = *reinterpret_cast<Int8Merge<D, kRows>*>(smem_raw);      // where the rings were
  // Behind an append of one token a sequence a block starts with what that append cannot write: the batch, and pages that do not hold the
  // newest token (rope_kv_write_int8 lets this kernel start only when all that came before it is done).  q and the newest page come later.
  // Behind anything else nothing is read before the kernels ahead are done: an append of several tokens writes the pages before
  // the newest too, and a kernel that lets its followers start before its own wait passes on what is not done yet.
  if (!p.beside && !p.after_append) grid_dependency_wait();
  const int seq = p.seq_index ? p.seq_index[blockIdx.z] : blockIdx.z;
  if (seq < 0) return;                          // a place of padding (the whole cluster's)
  const int q_begin = p.query_start_loc[seq];
  if (p.query_start_loc[seq + 1] == q_begin) return;
  const int split = blockIdx.x, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int groups = p.heads / p.kv_heads, hi = p.context_lens[seq];
  const int lo = first_visible(hi - 1, p.window);
  const int tile_lo = lo / kBlockN, tile_hi = (hi + kBlockN - 1) / kBlockN;
  const int per_split = (tile_hi - tile_lo + splits - 1) / splits;
  const int my_lo = tile_lo + split * per_split, my_hi = min(tile_hi, my_lo + per_split);
  const int my_groups = max(0, my_hi - my_lo);             // groups of 16 keys of this warp: one per tile of the block
  const int kpos_first = my_lo * kBlockN + warp * 16;      // of group i: kpos_first + 64 i
  const int* table = p.block_table + (size_t)seq * p.table_stride;

  // Of 32 groups at a time, a lane each, and of the 32 after them, which arrive meanwhile: the row where a group's keys lie (-1: none
  // that is visible) and the page's scales.
  struct Place { int row, scales; };
  auto place_of = [&](int i) {
    const int kpos0 = kpos_first + i * kBlockN;
    Place at{-1, 0};
    if (i < my_groups && kpos0 < hi && kpos0 + 16 > lo) {
      const int block = kpos0 / p.page_size, page = table[block];
      if (page >= 0 && page < p.num_pages) {
        at.scales = page * p.kv_heads + kvh;
        at.row = at.scales * p.page_size + (kpos0 - block * p.page_size);
      }
    }
    return at;
  };
  Place now = place_of(lane), next = my_groups > 32 ? place_of(32 + lane) : Place{-1, 0};
  const int settled = (hi - 1) / p.page_size * p.page_size;        // keys before this one lie in pages that the newest token does not
  const bool newest = kpos_first + lane * kBlockN >= settled;
  float k_scale = 0.f, log_v = 0.f;
  auto load_scales = [&]() {
    k_scale = p.k_scale[now.scales];
    log_v = fast_log2(p.v_scale[now.scales]);
  };
  if (now.row >= 0 && !newest) load_scales();
  float next_k = 0.f, next_v = 0.f;
  const unsigned ring = smem_addr(smem_raw) + (unsigned)warp * kRing * X * kGroupBytes + (unsigned)lane * 16;
  const signed char* const k_first = p.k_pool + g * D + t * 16;
  const signed char* const v_first = p.v_pool + 2 * t * D + g * (D / 8);
  // Asks for group i's keys and values.  Groups are asked for in their order, a turn's with one commit.
  auto request_one = [&](int i, int slot) {
    if ((i & 31) == 0 && i > 0) {
      now = next;
      k_scale = next_k;
      log_v = fast_log2(next_v);
      next = i + 32 < my_groups ? place_of(i + 32 + lane) : Place{-1, 0};
    } else if ((i & 31) == 16) {
      next_k = next.row >= 0 ? p.k_scale[next.scales] : 0.f;
      next_v = next.row >= 0 ? p.v_scale[next.scales] : 0.f;
    }
    const int row = __shfl_sync(0xffffffffu, now.row, i & 31);
    if (i < my_groups && row >= 0) {
      const signed char* k = k_first + (size_t)row * D;
      const signed char* v = v_first + (size_t)row * D;
      const unsigned at = ring + (unsigned)slot * kGroupBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + (h * (D / 64) + c) * 512), "l"(k + 8 * h * D + c * 64) : "memory");
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const signed char* from = v + ((q & 1) + (q >> 1) * 8) * D;
        if constexpr (D == 128) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + 2048 + q * 512), "l"(from) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at + 1024 + q * 256 - lane * 8), "l"(from) : "memory");
      }
    }
  };
  auto request = [&](int turn, int slot) {
#pragma unroll
    for (int x = 0; x < X; ++x) request_one(turn * X + x, slot * X + x);
    cp_async_commit();
  };
  const bool early = kpos_first + (min(my_groups, (kRing - 1) * X) - 1) * kBlockN < settled;      // (the same for the whole warp)
  if (early)
    for (int i = 0; i < kRing - 1; ++i) request(i, i);
  if (!p.beside) grid_dependency_wait();
  if (now.row >= 0 && newest) load_scales();
  if (!early)
    for (int i = 0; i < kRing - 1; ++i) request(i, i);

  // Q: head 8 j + g, the dimensions of this thread's place in K, word by word; what undoes its whole numbers (or its division) goes into
  // the factor of the head's scores.
  unsigned qb[NT][2][D / 16][2];        // kTwo: [piece][word of K][register]; else [h, l][pair of words of K][word], in half the room
  float factor[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = j * 8 + g;
    const T* src = (const T*)p.q + (size_t)q_begin * p.q_row_stride + (size_t)(kvh * groups + min(row, groups - 1)) * D;
    float x[D / 4];
    unsigned top = 0;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int e = 0; e < 16; e += Vec16<T>::N) {
        const Vec16<T> v = load16(src + c * 64 + t * 16 + e);
#pragma unroll
        for (int i = 0; i < Vec16<T>::N; ++i) {
          x[c * 16 + e + i] = v.get(i);
          top = max(top, abs_bits(v.get(i)));
        }
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const unsigned exponent = min(max(top >> 23, 1u), 253u);
    const float down = __uint_as_float((254u - exponent) << 23);      // 2^-e: the largest number times it lies in [1, 2)
    float up = __uint_as_float(exponent << 23);
    if constexpr (kTwo) {
#pragma unroll
      for (int w = 0; w < D / 16; ++w) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = x[w * 4 + i] * down;
        qb[j][0][w][0] = pack_half(y[0], y[2]);
        qb[j][0][w][1] = pack_half(y[1], y[3]);
        const float2 even = unpack_half(qb[j][0][w][0]), odd = unpack_half(qb[j][0][w][1]);
        qb[j][1][w][0] = pack_half(y[0] - even.x, y[2] - even.y);
        qb[j][1][w][1] = pack_half(y[1] - odd.x, y[3] - odd.y);
      }
    } else {
      const float largest = __uint_as_float(top) * down;              // NaN and infinity stay what they are, and so does `up` then
      const float steps = largest > 0.f ? kQuerySteps / largest : 0.f;
#pragma unroll
      for (int w = 0; w < D / 16; ++w) {
        unsigned high = 0, low = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int whole = __float2int_rn(x[w * 4 + i] * down * steps), h = (whole + 64) >> 7;
          high |= (unsigned)(h & 0xff) << (8 * i);
          low |= (unsigned)((whole - 128 * h) & 0xff) << (8 * i);
        }
        qb[j][0][w / 2][w & 1] = high;
        qb[j][1][w / 2][w & 1] = low;
      }
      up *= top > 0x7f800000u ? __uint_as_float(top) : largest / kQuerySteps;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      factor[j][e] = __shfl_sync(0xffffffffu, up, (2 * t + e) * 4) * p.scale * (kCapped ? 1.f / p.softcap : kLog2e);
  }
  const float cap = kCapped ? p.softcap * kLog2e : 0.f;

  float m[NT][2], r[NT][2], l[NT][2];
  float o[NT][D / 16][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[j][e] = r[j][e] = -INFINITY;
      l[j][e] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
  }

  // (what belongs to the groups that are multiplied, which lag behind those that are asked for)
  unsigned present = 0;
  float this_k = 0.f, this_v = 0.f;
  auto multiply = [&](int turn, int slot) {
    const int first = turn * X;
    if ((first & 31) == 0) {
      present = __ballot_sync(0xffffffffu, now.row >= 0);
      this_k = k_scale;
      this_v = log_v;
    }
    const unsigned there = present >> (first & 31) & ((1u << X) - 1u);
    if (there == 0) return;
    float page_k[X], page_v[X], s[X][NT][4];
    bool masked = there != (1u << X) - 1u;
#pragma unroll
    for (int x = 0; x < X; ++x) {
      page_k[x] = __shfl_sync(0xffffffffu, this_k, (first + x) & 31);
      page_v[x] = __shfl_sync(0xffffffffu, this_v, (first + x) & 31);
      const int kpos0 = kpos_first + (first + x) * kBlockN;
      masked |= kpos0 < lo || kpos0 + 16 > hi;
      const unsigned at = ring + (unsigned)(slot * X + x) * kGroupBytes;
      uint4 k[2][D / 64];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < D / 64; ++c) k[h][c] = shared16(at + (h * (D / 64) + c) * 512);
      if constexpr (kTwo) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][j][e] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            // A word of four serves one product: its bytes 0 and 2 are one register, 1 and 3 the other.
            const unsigned lo_w = word4(k[0][c], w), hi_w = word4(k[1][c], w);
            const unsigned a0 = halves_of(lo_w), a2 = halves_of(lo_w >> 8), a1 = halves_of(hi_w), a3 = halves_of(hi_w >> 8);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int piece = 0; piece < 2; ++piece)
                mma_f16(s[x][j], a0, a1, a2, a3, qb[j][piece][c * 4 + w][0], qb[j][piece][c * 4 + w][1]);
          }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          int high[4] = {0, 0, 0, 0}, low[4] = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int w = 0; w < 4; w += 2) {
              const unsigned a0 = word4(k[0][c], w), a1 = word4(k[1][c], w), a2 = word4(k[0][c], w + 1), a3 = word4(k[1][c], w + 1);
              mma_s8(high, a0, a1, a2, a3, qb[j][0][c * 2 + w / 2][0], qb[j][0][c * 2 + w / 2][1]);
              mma_s8(low, a0, a1, a2, a3, qb[j][1][c * 2 + w / 2][0], qb[j][1][c * 2 + w / 2][1]);
            }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][j][e] = (float)(high[e] * 128 + low[e]);      // at most 128 * 127 * 16256 < 2^28
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[x][j][e] *= factor[j][e & 1] * page_k[x];
          if constexpr (kCapped) s[x][j][e] = cap * fast_tanh(s[x][j][e]);
        }
    }
    if (masked) {
#pragma unroll
      for (int x = 0; x < X; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kpos = kpos_first + (first + x) * kBlockN + g + 8 * h;
          if (kpos < lo || kpos >= hi || !(there >> x & 1)) {
#pragma unroll
            for (int j = 0; j < NT; ++j) s[x][j][2 * h] = s[x][j][2 * h + 1] = -INFINITY;
          }
        }
    }
    // The largest of this thread's scores of a head, and the largest with its page's scale of values.
    auto largest = [&](int j, int e, float& plain, float& scaled) {
      plain = scaled = -INFINITY;
#pragma unroll
      for (int x = 0; x < X; ++x) {
        const float top = fmaxf(s[x][j][e], s[x][j][e + 2]);
        plain = fmaxf(plain, top);
        scaled = fmaxf(scaled, top + page_v[x]);
      }
    };
    bool grows = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float plain, scaled;
        largest(j, e, plain, scaled);
        grows |= plain > m[j][e] + 16.f || scaled > r[j][e] + 15.f;
      }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float plain, scaled;
          largest(j, e, plain, scaled);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            plain = fmaxf(plain, __shfl_xor_sync(0xffffffffu, plain, x));
            scaled = fmaxf(scaled, __shfl_xor_sync(0xffffffffu, scaled, x));
          }
          const float m_new = fmaxf(m[j][e], plain), r_new = fmaxf(r[j][e], scaled - 8.f);
          const float keep_l = m_new == -INFINITY ? 1.f : fast_exp2(m[j][e] - m_new);
          const float keep_o = r_new == -INFINITY ? 1.f : fast_exp2(r[j][e] - r_new);
          m[j][e] = m_new;
          r[j][e] = r_new;
          l[j][e] *= keep_l;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[j][d][e] *= keep_o;
            o[j][d][e + 2] *= keep_o;
          }
        }
    }
    unsigned pb[X][NT][kPieces][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float m_use[2], r_use[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m_use[e] = m[j][e] == -INFINITY ? 0.f : m[j][e];
        r_use[e] = r[j][e] == -INFINITY ? 0.f : r[j][e];
      }
#pragma unroll
      for (int x = 0; x < X; ++x) {
        // exp2(s + log2 s_v - r) = exp2(s - m) * exp2(log2 s_v + m - r), the second factor the page's.  (At most 2^126: a page whose scale
        // is 2^120 times the others' has lost bits before.)
        float w[4], page[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float up = page_v[x] + (m_use[e] - r_use[e]);
          page[e] = fast_exp2(up > 126.f ? 126.f : up);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float weight = fast_exp2(s[x][j][e] - m_use[e & 1]);
          l[j][e & 1] += weight;
          w[e] = weight * page[e & 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned packed = pack_half(w[2 * h], w[2 * h + 1]);
          pb[x][j][0][h] = turned(packed);
          if constexpr (kTwo) {
            const float2 rounded = unpack_half(packed);
            pb[x][j][1][h] = turned(pack_half(w[2 * h] - rounded.x, w[2 * h + 1] - rounded.y));
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const unsigned at = ring + (unsigned)(slot * X + x) * kGroupBytes;
      uint4 v[4];             // (D 64: two words of each)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (D == 128) {
          v[q] = shared16(at + 2048 + q * 512);
        } else {
          const uint2 two = shared8(at + 1024 + q * 256 - lane * 8);
          v[q].x = two.x; v[q].y = two.y;
        }
      }
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        const int w = n / 2;                                 // this tile's two dimensions: two bytes of word w
        const unsigned even = n & 1 ? 0x6622u : 0x4400u, odd = n & 1 ? 0x7733u : 0x5511u;
        const unsigned x0 = word4(v[0], w), x1 = word4(v[1], w), x2 = word4(v[2], w), x3 = word4(v[3], w);
        const unsigned a0 = halves_of(__byte_perm(x0, x1, even)), a1 = halves_of(__byte_perm(x0, x1, odd));
        const unsigned a2 = halves_of(__byte_perm(x2, x3, even)), a3 = halves_of(__byte_perm(x2, x3, odd));
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int piece = 0; piece < kPieces; ++piece) mma_f16(o[j][n], a0, a1, a2, a3, pb[x][j][piece][0], pb[x][j][piece][1]);
      }
    }
  };
  int slot = 0;
  for (int turn = 0; turn * X < my_groups; ++turn) {
    request(turn + kRing - 1, slot == 0 ? kRing - 1 : slot - 1);     // in the place of the turn before this one
    cp_async_wait<kRing - 1>();
    multiply(turn, slot);
    slot = slot == kRing - 1 ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  __syncthreads();          // the rings are free
  grid_launch_dependents();

  // The warps' states.  Thread (g, t) holds, of heads 2t and 2t + 1 of each tile, the dimensions g D/8 ...
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], x);
      const int row = j * 8 + 2 * t + e;
      const float back = r[j][e] == -INFINITY ? 1.f : fast_exp2(r[j][e] - m[j][e]);      // from its own reference to the denominator's
      if (row < groups) {
        float4* dst = reinterpret_cast<float4*>(&merge.os[warp][row][g * (D / 8)]);
#pragma unroll
        for (int d = 0; d < D / 16; d += 2)
          dst[d / 2] = make_float4(o[j][d][e] * back, o[j][d][e + 2] * back, o[j][d + 1][e] * back, o[j][d + 1][e + 2] * back);
        if (g == 0) {
          merge.ms[warp][row] = m[j][e];
          merge.ls[warp][row] = l[j][e];
        }
      }
    }
  __syncthreads();
  auto store = [&](int row, int d4, float4 v) {
    T* dst = (T*)p.out + (size_t)q_begin * p.out_row_stride + (size_t)(kvh * groups + row) * D + d4 * 4;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = v;
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
  };
  for (int item = threadIdx.x; item < groups * (D / 4); item += kWarps * 32) {
    const int row = item / (D / 4), d4 = item % (D / 4);
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge.ms[w][row]);
    float denom = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = merge.ms[w][row], weight = mw == -INFINITY ? 0.f : exp2f(mw - top);
      const float4 v = reinterpret_cast<const float4*>(merge.os[w][row])[d4];
      if (mw == -INFINITY && merge.ls[w][row] == 0.f) continue;       // a warp that saw no key
      denom += weight * merge.ls[w][row];
      acc.x += weight * v.x; acc.y += weight * v.y; acc.z += weight * v.z; acc.w += weight * v.w;
    }
    if (splits == 1) {
      if (p.sink != nullptr) denom += exp2f(p.sink[kvh * groups + row] * kLog2e - top);
      const float inv = denom == 0.f ? 0.f : 1.f / denom;
      store(row, d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    } else {
      const float inv = denom == 0.f ? 0.f : 1.f / denom;
      reinterpret_cast<float4*>(merge.mine[row])[d4] = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (d4 == 0) merge.lse[row] = denom == 0.f ? -INFINITY : top + log2f(denom);
    }
  }
  if (splits == 1) return;
  cluster_sync_all();                                    // every block's result is in place (release / acquire)
  auto remote = [&](const float* local, int rank) {      // the same place in the shared memory of block `rank`
    unsigned addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(local)), "r"(rank));
    return addr;
  };
  for (int item = split * (kWarps * 32) + threadIdx.x; item < groups * (D / 4); item += splits * (kWarps * 32)) {
    const int row = item / (D / 4), d4 = item % (D / 4);
    float w[8];
    float4 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < splits) {
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w[x]) : "r"(remote(&merge.lse[row], x)));
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[x].x), "=f"(v[x].y), "=f"(v[x].z), "=f"(v[x].w) : "r"(remote(&merge.mine[row][d4 * 4], x)));
      }
    float top = -INFINITY, denom = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < splits) top = fmaxf(top, w[x]);
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < splits && w[x] != -INFINITY) {
        const float weight = exp2f(w[x] - top);
        denom += weight;
        acc.x += weight * v[x].x; acc.y += weight * v[x].y; acc.z += weight * v[x].z; acc.w += weight * v[x].w;
      }
    if (p.sink != nullptr) denom += exp2f(p.sink[kvh * groups + row] * kLog2e - top);
    const float inv = denom == 0.f ? 0.f : 1.f / denom;
    store(row, d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
  cluster_sync_all();                                    // nobody leaves while another reads
}

template <typename T, int D, int NT, bool kCapped>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? (sizeof(T) == 2 || D == 64 ? 4 : 3) : 2)
attention_int8_kernel(const Int8AttnParams p, int splits) {
  attend<T, D, NT, kCapped>(p, splits);
  // What follows waits for this kernel, and through it for the one beside it.
  if (p.beside) grid_dependency_wait();
}

template <typename T, int D, int NT> constexpr size_t attention_smem() {
  constexpr size_t rings = (size_t)kWarps * kRing * kTurn<T, D> * 16 * D * 2;
  return rings > sizeof(Int8Merge<D, NT * 8>) ? rings : sizeof(Int8Merge<D, NT * 8>);
}

template <typename T, int D, int NT, bool kCapped>
static int launch_attention(const Int8AttnParams& p, int num_seqs, int splits, cudaStream_t stream) {
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(attention_int8_kernel<T, D, NT, kCapped>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)attention_smem<T, D, NT>());
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(splits, p.kv_heads, num_seqs);
  config.blockDim = dim3(kWarps * 32);
  config.dynamicSmemBytes = attention_smem<T, D, NT>();
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  int count = 0;
  if (pdl_enabled(num_seqs)) {
    attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[count++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (splits > 1) {
    attributes[count].id = cudaLaunchAttributeClusterDimension;
    attributes[count].val.clusterDim.x = splits;
    attributes[count].val.clusterDim.y = 1;
    attributes[count++].val.clusterDim.z = 1;
  }
  config.attrs = attributes;
  config.numAttrs = count;
  return (int)cudaLaunchKernelEx(&config, attention_int8_kernel<T, D, NT, kCapped>, p, splits);
}

template <typename T, int D>
static int launch_heads(const Int8AttnParams& p, int num_seqs, int splits, cudaStream_t stream) {
  const bool capped = p.softcap > 0.f;
  if (p.heads / p.kv_heads <= 8)
    return capped ? launch_attention<T, D, 1, true>(p, num_seqs, splits, stream) : launch_attention<T, D, 1, false>(p, num_seqs, splits, stream);
  return capped ? launch_attention<T, D, 2, true>(p, num_seqs, splits, stream) : launch_attention<T, D, 2, false>(p, num_seqs, splits, stream);
}

template <typename T, int D, int NT>
static int capacity() {
  static int blocks = 0;
  if (blocks) return blocks;
  int device = 0, sms = 0, per_sm = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      cudaFuncSetAttribute(attention_int8_kernel<T, D, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attention_smem<T, D, NT>()) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attention_int8_kernel<T, D, NT, false>, kWarps * 32, attention_smem<T, D, NT>()) != cudaSuccess)
    return 0;
  return blocks = sms * per_sm;
}

}  // namespace li

using namespace li;

// Whether li_attention_int8 takes these sizes.
LI_EXPORT int li_attention_int8_supports(int heads, int kv_heads, int head_dim, int page_size) {
  if (kv_heads < 1 || heads % kv_heads || heads / kv_heads > 16 || heads < 1) return 0;
  return (head_dim == 64 || head_dim == 128) && page_size >= 16 && page_size % 16 == 0;
}

// Blocks of the kernel that the device holds at once (0: the query failed).
LI_EXPORT int li_attention_int8_capacity(int dtype, int head_dim, int groups) {
  if (dtype == kFloat32) {
    if (head_dim == 64) return groups <= 8 ? capacity<float, 64, 1>() : capacity<float, 64, 2>();
    return groups <= 8 ? capacity<float, 128, 1>() : capacity<float, 128, 2>();
  }
  if (head_dim == 64) return groups <= 8 ? capacity<bf16, 64, 1>() : capacity<bf16, 64, 2>();
  return groups <= 8 ? capacity<bf16, 128, 1>() : capacity<bf16, 128, 2>();
}

struct AttentionInt8Args {
  long long dtype;          // of q and out
  const void* q;
  long long q_row_stride;
  void* out;
  long long out_row_stride;
  const void *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int* block_table;
  long long table_stride;
  const int *query_start_loc, *context_lens, *seq_index;
  long long num_seqs, heads, kv_heads, head_dim, page_size, num_pages;
  double scale;
  long long window;
  double softcap;
  const float* sink;
  long long splits;         // 1, 2, 4 or 8 blocks share a sequence's keys
  long long beside;         // the kernel ahead on the stream is the same step's li_attention_int8_prompt
  long long after_append;   // the kernel ahead on the stream is li_rope_kv_write_int8 and writes one token at most of each of these sequences
  cudaStream_t stream;
};

// Every launched sequence brings at most one token.
LI_EXPORT int li_attention_int8(const AttentionInt8Args* a) {
  const int num_seqs = (int)a->num_seqs, splits = (int)a->splits;
  if (num_seqs == 0) return 0;
  if (!li_attention_int8_supports((int)a->heads, (int)a->kv_heads, (int)a->head_dim, (int)a->page_size) || a->kv_heads > 65535 || num_seqs > 65535)
    return LI_ERR_UNSUPPORTED;
  if (splits != 1 && splits != 2 && splits != 4 && splits != 8) return LI_ERR_UNSUPPORTED;
  if (a->num_pages * a->kv_heads * a->page_size > 0x7fffffffL) return LI_ERR_UNSUPPORTED;
  const size_t size = a->dtype == kFloat32 ? 4 : 2;
  if (!aligned16(a->q) || a->q_row_stride * size % 16 || !aligned16(a->out) || a->out_row_stride * size % 16 || !aligned16(a->k_pool) ||
      !aligned16(a->v_pool))
    return LI_ERR_ALIGNMENT;
  Int8AttnParams p{a->q, (int)a->q_row_stride, a->out, (int)a->out_row_stride, (const signed char*)a->k_pool, (const signed char*)a->v_pool,
                   a->k_scale, a->v_scale, a->block_table, (int)a->table_stride, a->query_start_loc, a->context_lens, a->seq_index,
                   (int)a->heads, (int)a->kv_heads, (int)a->page_size, (int)a->num_pages, (float)a->scale, (int)a->window,
                   (float)a->softcap, a->sink, a->beside != 0, a->after_append != 0};
  if (a->dtype == kFloat32)
    return a->head_dim == 64 ? launch_heads<float, 64>(p, num_seqs, splits, a->stream) : launch_heads<float, 128>(p, num_seqs, splits, a->stream);
  return a->head_dim == 64 ? launch_heads<bf16, 64>(p, num_seqs, splits, a->stream) : launch_heads<bf16, 128>(p, num_seqs, splits, a->stream);
}
