// A paged cache whose keys and values are held in 8 bits, with one scale for each page and KV head (and one for the keys, one for
// the values): appending to it with the rotary encoding on the way, and reading its pages back.
//
//   pool [pages][kv_heads][page_size][head_dim] int8, scale [pages][kv_heads] float
//
// Appending.  Token t of the batch stands at position p of sequence s and goes to slot p % page_size of page
// block_table[s][p / page_size]; a sequence's tokens lie in the batch one behind the other, at consecutive positions.  The
// tokens of one sequence that land in the same page are one item: they need the scale max |x| * (1/127), the page keeps its scale if
// it is as large, and otherwise grows it (grown_scale, int8.cuh) and rounds the whole numbers of the tokens before them
// again.  Where the first of them takes slot 0 the page is new: whatever it held is forgotten, its scale too.  Tokens behind the last
// of them count as not there.  An item belongs to one block, so nothing depends on an order between blocks.
#include "int8.cuh"

namespace li {

constexpr int kAppendWarps = 8;

struct AppendParams {
  const void* qkv;          // rows [q heads | k heads | v heads]
  size_t row_stride;
  void* q_out;              // rotated q, a row a token
  size_t q_out_stride;
  const int* positions;
  const int* seq_of_token;  // negative: a row of padding
  const int* block_table;
  int table_stride;
  signed char* pool[2];     // keys, values
  float* scale[2];
  const float* inv_freq;    // null: nothing is rotated
  int tokens, heads, kv_heads, head_dim, rotary_dim, page_size, num_pages;
  float cs_scale;
};

struct AppendItem { int count, page, slot; };       // an item's tokens (0: none starts here), its page (-1: nothing is stored), first slot
// Whether token t (below p.tokens) does not follow the one before it in the batch within the same page.
__device__ __forceinline__ bool starts_item(const AppendParams& p, int t, int pos, int seq) {
  return t == 0 || pos % p.page_size == 0 || p.seq_of_token[t - 1] != seq || p.positions[t - 1] != pos - 1;
}
__device__ __forceinline__ int page_of_token(const AppendParams& p, int pos, int seq) {
  if (seq < 0 || p.num_pages == 0) return -1;
  const int page = p.block_table[(size_t)seq * p.table_stride + pos / p.page_size];
  return page < p.num_pages ? page : -1;
}

// Sixteen numbers of a token's head as they lie in memory: where it is rotated, dimensions 8u ... and half + 8u ...; behind the rotated
// ones, 16 neighbours.  (They wait in that form, bfloat16 in half the registers, and are rotated where they are used.)
template <typename T> struct Sixteen {
  static constexpr int N = Vec16<T>::N;
  Vec16<T> a[8 / N], b[8 / N];
  // The first dimensions of either half.
  __device__ __forceinline__ static int first(int u, int half) { return 8 * u < half ? 8 * u : 16 * u; }      // (16 u = 2 half + 16 (u - half / 8))
  __device__ __forceinline__ static int second(int u, int half) { return 8 * u < half ? half + 8 * u : 16 * u + 8; }
  __device__ __forceinline__ void fetch(const T* head, int u, int half) {
    const int at = first(u, half), bt = second(u, half);
#pragma unroll
    for (int e = 0; e < 8 / N; ++e) {
      a[e] = load16(head + at + e * N);
      b[e] = load16(head + bt + e * N);
    }
  }
  // The numbers, rotated: x of the first half, y of the second.
  __device__ __forceinline__ void turned(int u, int half, const float* cosv, float (&x)[8], float (&y)[8]) const {
#pragma unroll
    for (int e = 0; e < 8 / N; ++e) {
      unpack16(a[e], x + e * N);
      unpack16(b[e], y + e * N);
    }
    if (8 * u < half) {
      float c[8], s[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(cosv + 8 * u + e);
        *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(cosv + half + 8 * u + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = x[e], q = y[e];
        x[e] = rotate_lo(p, q, c[e], s[e]);
        y[e] = rotate_hi(p, q, c[e], s[e]);
      }
    }
  }
  __device__ __forceinline__ unsigned largest(int u, int half, const float* cosv) const {
    if constexpr (N == 8) {
      if (8 * u >= half) {                  // not rotated: the magnitudes of bfloat16 as whole numbers, two at a time
        const unsigned w[8] = {a[0].raw.x, a[0].raw.y, a[0].raw.z, a[0].raw.w, b[0].raw.x, b[0].raw.y, b[0].raw.z, b[0].raw.w};
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
        return max(top << 16, top & 0xffff0000u);
      }
    }
    float x[8], y[8];
    turned(u, half, cosv, x, y);
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, max(abs_bits(x[e]), abs_bits(y[e])));
    return top;
  }
  __device__ __forceinline__ void store(T* head, int u, int half, const float* cosv) const {
    float x[8], y[8];
    turned(u, half, cosv, x, y);
    const int at = first(u, half), bt = second(u, half);
#pragma unroll
    for (int e = 0; e < 8 / N; ++e) {
      Vec16<T> v, w;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v.set(i, x[e * N + i]);
        w.set(i, y[e * N + i]);
      }
      store16(head + at + e * N, v);
      store16(head + bt + e * N, w);
    }
  }
  __device__ __forceinline__ void quantise(signed char* head, int u, int half, const float* cosv, float scale, float inverse, bool plain) const {
    float x[8], y[8];
    turned(u, half, cosv, x, y);
    *reinterpret_cast<uint2*>(head + first(u, half)) = make_uint2(quantised4(x, scale, inverse, plain), quantised4(x + 4, scale, inverse, plain));
    *reinterpret_cast<uint2*>(head + second(u, half)) = make_uint2(quantised4(y, scale, inverse, plain), quantised4(y + 4, scale, inverse, plain));
  }
};

// Every run of up to `chunk` tokens has three blocks (blockIdx.y): one for its q heads, sixteen numbers a thread at a time, one for the keys
// and one for the values of the items that start in it, whose (item, head)s the warps take in turn.  A warp holds a page's new numbers of a head in
// registers between the maximum and the rounding where they are at most 128 sixteens (16 tokens of 128 dimensions), and loads them
// again where they are more.  Cosines and sines are computed once for all heads.  Where items start is found for all tokens at once
// (a loop over each item's tokens in memory took 8 us).  Bound by memory where heads are many.  Where they are few, by the chain of a block
// (batch, table, numbers, largest, scale), so that blocks of four warps, of which more run at once, take it (7,144 tokens, 2 heads on 1 of 64:
// 15 us with the read-back, 23 with eight warps).
constexpr int kMaxChunk = 16, kMaxPage = 1024;
constexpr int kHeldSixteens = 4;         // a lane

template <typename T, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, (sizeof(T) == 2 ? 24 : 16) / kWarps) rope_kv_write_int8_kernel(const AppendParams p, int chunk) {
  extern __shared__ float angles[];      // [tokens][2][half]
  __shared__ AppendItem items[kMaxChunk];
  __shared__ int several[kMaxChunk], single[kMaxChunk];       // the tokens that items of more than one start at, and of one
  __shared__ unsigned starts[(kMaxChunk + kMaxPage + kWarps * 32 - 1) / (kWarps * 32) * kWarps];
  __shared__ int first_pos[kMaxChunk + kMaxPage];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, role = blockIdx.y;
  const int half = p.inv_freq != nullptr ? p.rotary_dim / 2 : 0, D = p.head_dim, units = D / 16;
  const int t0 = blockIdx.x * chunk, mine = min(chunk, p.tokens - t0);
  grid_dependency_wait();
  // Only now may the kernel behind start: what came before this launch is done, and the attention of single tokens may read, while this one
  // still writes, the pages that it does not touch.
  grid_launch_dependents();
  const T* const rows = (const T*)p.qkv + (size_t)t0 * p.row_stride;
  int from = 0, reach = mine;             // tokens whose angles are needed
  __shared__ int numbers[2];              // of either
  if (role > 0) {
    const int window = min(chunk + p.page_size, p.tokens - t0);
    int my_pos = 0, my_seq = -1;
    bool my_start = false;
    for (int k0 = 0; k0 < window; k0 += kWarps * 32) {
      const int k = k0 + threadIdx.x, t = t0 + k;
      int pos = 0, seq = -1;
      bool start = true;
      if (k < window) {
        pos = p.positions[t];
        seq = p.seq_of_token[t];
        start = starts_item(p, t, pos, seq);
        first_pos[k] = pos;
      }
      if (k0 == 0) { my_pos = pos; my_seq = seq; my_start = start; }
      const unsigned mask = __ballot_sync(0xffffffffu, start);      // (what lies behind the batch starts as well: it ends the item before)
      if (lane == 0) starts[k / 32] = mask;
    }
    __syncthreads();
    auto next_start = [&](int k) {        // the first start behind token k, at most `window`
      int w = (k + 1) >> 5;
      unsigned mask = starts[w] & (0xffffffffu << ((k + 1) & 31));
      while (mask == 0 && (w + 1) * 32 < window) mask = starts[++w];
      return mask == 0 ? window : min(window, w * 32 + __ffs(mask) - 1);
    };
    if (warp == 0) {                      // (mine is at most 16)
      AppendItem item{0, -1, my_pos % p.page_size};
      if (lane < mine && my_start) {
        item.page = page_of_token(p, my_pos, my_seq);
        if (item.page >= 0) item.count = next_start(lane) - lane;
      }
      const unsigned more = __ballot_sync(0xffffffffu, item.count > 1), one = __ballot_sync(0xffffffffu, item.count == 1), below = (1u << lane) - 1u;
      if (lane < mine) items[lane] = item;
      if (item.count > 1) several[__popc(more & below)] = lane;
      if (item.count == 1) single[__popc(one & below)] = lane;
      if (lane == 0) {
        numbers[0] = __popc(more);
        numbers[1] = __popc(one);
      }
    }
    const unsigned among = starts[0] & ((1u << mine) - 1u);
    if (among == 0) return;               // (the whole block: all its tokens follow)
    from = __ffs(among) - 1;
    reach = next_start(mine - 1);
  } else if (threadIdx.x < mine) {
    first_pos[threadIdx.x] = p.positions[t0 + threadIdx.x];
  }
  __syncthreads();
  if (role < 2) {
    for (int i = from * half + threadIdx.x; i < reach * half; i += blockDim.x) {
      const int n = i / half, j = i - n * half;
      const float angle = __fmul_rn((float)first_pos[n], p.inv_freq[j]);
      float s, c;
      sincosf(angle, &s, &c);             // (the same bits as sinf and cosf for every angle up to 2^23)
      angles[n * 2 * half + j] = c * p.cs_scale;
      angles[n * 2 * half + half + j] = s * p.cs_scale;
    }
    __syncthreads();
  }
  if (role == 0) {
    if (half == 0 && p.q_out == p.qkv) return;
    // A thread keeps its place in the heads and takes the tokens in turn, four at a time, loads first; where the heads are fewer than the
    // threads, several tokens go side by side.
    constexpr int kAtOnce = sizeof(T) == 2 ? 4 : 2, kThreads = kWarps * 32;
    const int per_token = p.heads * units, beside = per_token < kThreads ? kThreads / per_token : 1;
    const int n_first = beside > 1 ? threadIdx.x / per_token : 0;
    if (n_first >= beside) return;
    T* const out = (T*)p.q_out + (size_t)t0 * p.q_out_stride;
    for (int place = threadIdx.x - n_first * per_token; place < per_token; place += kThreads) {
      const int h = place / units, u = place - h * units;
      for (int n = n_first; n < mine; n += kAtOnce * beside) {
        Sixteen<T> x[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (n + k * beside < mine) x[k].fetch(rows + (n + k * beside) * p.row_stride + h * D, u, half);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          if (n + k * beside < mine)
            x[k].store(out + (n + k * beside) * p.q_out_stride + h * D, u, half, angles + (n + k * beside) * 2 * half);
      }
      if (beside > 1) break;
    }
    return;
  }
  const int which = role - 1, turned = which == 0 ? half : 0;
  const int side = 32 / units, beside = lane / units, u = lane - beside * units;      // tokens that lie side by side in a warp
  const auto grow = [&](signed char* out, int first, int step, int vectors, float old, float scale) {
    // The tokens that are there, with the larger scale.
    const float ratio = scale_holds(scale) ? __fdiv_rn(old, scale) : 0.f;
    for (int v = first; v < vectors; v += step) {
      uint4 raw = reinterpret_cast<const uint4*>(out)[v];
      unsigned* words = reinterpret_cast<unsigned*>(&raw);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) r |= (unsigned)(requantised((signed char)(words[k] >> (8 * e)), ratio) & 0xff) << (8 * e);
        words[k] = r;
      }
      reinterpret_cast<uint4*>(out)[v] = raw;
    }
  };
  // Items of one token: as many heads side by side in a warp as fit (64 single tokens beside 2,000 of a portion, 32 heads on 8 of 128:
  // 34 us with the read-back a head at a time, 24 so).
  const int sets = (p.kv_heads + side - 1) / side;
  for (int i = warp; i < numbers[1] * sets; i += kWarps) {
    const int n0 = single[i / sets], h = i % sets * side + beside;
    if (beside >= side || h >= p.kv_heads) continue;
    const AppendItem item = items[n0];
    float* const at = p.scale[which] + (size_t)item.page * p.kv_heads + h;
    signed char* const out = p.pool[which] + ((size_t)item.page * p.kv_heads + h) * p.page_size * D;
    const float old = item.slot > 0 ? *at : 0.f;
    const float* const cosv = angles + n0 * 2 * half;
    Sixteen<T> x;
    x.fetch(rows + (size_t)n0 * p.row_stride + (size_t)(p.heads + which * p.kv_heads + h) * D, u, turned);
    const unsigned lanes = ((units == 32 ? 0u : 1u << units) - 1u) << (beside * units);
    const float scale = grown_scale(old, scale_of(__reduce_max_sync(lanes, x.largest(u, turned, cosv))));
    const bool plain = scale_plain(scale);
    x.quantise(out + item.slot * D, u, turned, cosv, scale, plain ? __frcp_rn(scale) : 0.f, plain);
    if (item.slot > 0 && scale != old) grow(out, u, units, item.slot * units, old, scale);
    if (u == 0) *at = scale;
  }
  __syncwarp();
  int k_next = warp / p.kv_heads, h_next = warp % p.kv_heads;
  for (; k_next < numbers[0];) {
    const int n0 = several[k_next], h = h_next;
    for (h_next += kWarps; h_next >= p.kv_heads; h_next -= p.kv_heads) ++k_next;
    const AppendItem item = items[n0];
    {
      float* const at = p.scale[which] + (size_t)item.page * p.kv_heads + h;
      signed char* const out = p.pool[which] + ((size_t)item.page * p.kv_heads + h) * p.page_size * D;
      const float old = item.slot > 0 ? *at : 0.f;
      // This lane's numbers: place u of every token lane / units + k * side of the item.
      const T* const src = rows + (size_t)(n0 + beside) * p.row_stride + (size_t)(p.heads + which * p.kv_heads + h) * D;
      const float* const cosv = angles + (n0 + beside) * 2 * half;
      signed char* const dst = out + (item.slot + beside) * D;
      const int mine_of_item = beside < side ? (item.count - beside + side - 1) / side : 0;
      Sixteen<T> held[kHeldSixteens], x;
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < kHeldSixteens; ++k)
        if (k < mine_of_item) held[k].fetch(src + k * side * p.row_stride, u, turned);
#pragma unroll
      for (int k = 0; k < kHeldSixteens; ++k)
        if (k < mine_of_item) top = max(top, held[k].largest(u, turned, cosv + k * side * 2 * half));
      for (int k = kHeldSixteens; k < mine_of_item; ++k) {
        x.fetch(src + k * side * p.row_stride, u, turned);
        top = max(top, x.largest(u, turned, cosv + k * side * 2 * half));
      }
      const float scale = grown_scale(old, scale_of(warp_max_bits(top)));
      const bool plain = scale_plain(scale);
      const float inverse = plain ? __frcp_rn(scale) : 0.f;
#pragma unroll
      for (int k = 0; k < kHeldSixteens; ++k)
        if (k < mine_of_item) held[k].quantise(dst + k * side * D, u, turned, cosv + k * side * 2 * half, scale, inverse, plain);
      for (int k = kHeldSixteens; k < mine_of_item; ++k) {
        x.fetch(src + k * side * p.row_stride, u, turned);
        x.quantise(dst + k * side * D, u, turned, cosv + k * side * 2 * half, scale, inverse, plain);
      }
      if (item.slot > 0 && scale != old) grow(out, lane, 32, item.slot * units, old, scale);
      if (lane == 0) *at = scale;
    }
  }
}

// The same for a rotary width that is no multiple of 16, and for pages whose tokens' cosines and sines fit no shared memory: a block a token, a
// number at a time.  kAngles: they do fit; else each is computed where it is used.
template <bool kAngles, typename T>
__device__ __forceinline__ float rotated(const AppendParams& p, const T* row, int j, int half, int pos, const float* cosv) {
  if (j >= 2 * half) return to_float(row[j]);
  const int i = j < half ? j : j - half;
  float c, s;
  if constexpr (kAngles) {
    c = cosv[i];
    s = cosv[half + i];
  } else {
    const float angle = __fmul_rn((float)pos, p.inv_freq[i]);
    c = cosf(angle) * p.cs_scale;
    s = sinf(angle) * p.cs_scale;
  }
  const float a = to_float(row[i]), b = to_float(row[i + half]);
  return j < half ? rotate_lo(a, b, c, s) : rotate_hi(a, b, c, s);
}

template <typename T, bool kAngles>
__global__ void __launch_bounds__(kAppendWarps * 32) rope_kv_write_int8_odd_kernel(const AppendParams p) {
  extern __shared__ float shared[];      // kAngles: cosines and sines of the item's positions: [page_size][2][half]
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = p.inv_freq != nullptr ? p.rotary_dim / 2 : 0, D = p.head_dim;
  grid_dependency_wait();
  grid_launch_dependents();
  const int pos = p.positions[t], seq = p.seq_of_token[t], slot = pos % p.page_size;
  const int page = starts_item(p, t, pos, seq) ? page_of_token(p, pos, seq) : -1;
  int count = page >= 0 ? 1 : 0;
  if (page >= 0)
    while (t + count < p.tokens && !starts_item(p, t + count, p.positions[t + count], p.seq_of_token[t + count])) ++count;
  const int turns = max(count, 1);
  if (kAngles) {
    for (int i = threadIdx.x; i < turns * half; i += blockDim.x) {
      const int n = i / half, j = i - n * half;
      const float angle = __fmul_rn((float)(pos + n), p.inv_freq[j]);
      shared[n * 2 * half + j] = cosf(angle) * p.cs_scale;
      shared[n * 2 * half + half + j] = sinf(angle) * p.cs_scale;
    }
    __syncthreads();
  }
  const T* row0 = (const T*)p.qkv + (size_t)t * p.row_stride;
  T* q_out = (T*)p.q_out + (size_t)t * p.q_out_stride;
  // (q may be rotated in place: a warp reads a head whole before it writes it, at most 512 dimensions of it)
  for (int h = warp; h < p.heads; h += kAppendWarps) {
    const T* src = row0 + (size_t)h * D;
    T* dst = q_out + (size_t)h * D;
    float r[16];
    for (int i = 0, j = lane; j < D; j += 32, ++i) r[i] = rotated<kAngles>(p, src, j, half, pos, shared);
    __syncwarp();
    for (int i = 0, j = lane; j < D; j += 32, ++i) dst[j] = from_float<T>(r[i]);
  }
  if (page < 0) return;
  for (int item = warp; item < 2 * p.kv_heads; item += kAppendWarps) {
    const int which = item / p.kv_heads, h = item - which * p.kv_heads;
    const T* src = row0 + (size_t)(p.heads + which * p.kv_heads + h) * D;
    const int turned = which == 0 ? half : 0;
    unsigned top = 0;
    for (int n = 0; n < count; ++n)
      for (int j = lane; j < D; j += 32)
        top = max(top, abs_bits(rotated<kAngles>(p, src + n * p.row_stride, j, turned, pos + n, shared + n * 2 * half)));
    const float need = scale_of(warp_max_bits(top));
    float* at = p.scale[which] + (size_t)page * p.kv_heads + h;
    const float old = slot > 0 ? *at : 0.f, scale = grown_scale(old, need);
    signed char* out = p.pool[which] + ((size_t)page * p.kv_heads + h) * p.page_size * D;
    if (slot > 0 && scale != old) {
      const float ratio = scale_holds(scale) ? __fdiv_rn(old, scale) : 0.f;
      for (int j = lane; j < slot * D; j += 32) out[j] = (signed char)requantised(out[j], ratio);
    }
    const bool holds = scale_holds(scale);
    for (int n = 0; n < count; ++n)
      for (int j = lane; j < D; j += 32)
        out[(slot + n) * D + j] = (signed char)quantised(rotated<kAngles>(p, src + n * p.row_stride, j, turned, pos + n, shared + n * 2 * half), scale, holds);
    __syncwarp();
    if (lane == 0) *at = scale;
  }
}

struct ReadParams {
  const signed char* pool[2];
  const float* scale[2];
  const int* block_table;
  int table_stride;
  const int* lens;
  const int* row_index;     // optional: which row of block_table, lens and query_start_loc the i-th row read is (negative: none)
  const int* query_start_loc;   // optional: only what a row's newest queries can see is read, by `window` and `keep_first`
  int window, keep_first;
  int* table_out;           // optional: the table of what is read, block b of row r in page r * blocks + b of the outputs
  void* out[2];             // [rows][blocks][kv_heads][page_size][head_dim]
  int blocks, kv_heads, head_dim, page_size, num_pages;
};

// A block a share of a (row, block of the row, keys or values), 16 numbers a thread at a time.  Bound by memory: a byte in and two or
// four out a number.  (Four of them a thread: 17 us for 520 pages of 8 heads, 16 tokens and 128 dimensions, 23 with one a thread.)
template <typename T>
__global__ void __launch_bounds__(256) read_pages_int8_kernel(const ReadParams p) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.x, which = blockIdx.y & 1, part = blockIdx.y >> 1, i = blockIdx.z;
  const int row = p.row_index != nullptr ? p.row_index[i] : i;
  if (row < 0) return;
  const int len = p.lens[row], first = b * p.page_size;
  int page = p.block_table[(size_t)row * p.table_stride + b];
  if (page >= p.num_pages || first >= len) page = -1;
  if (p.query_start_loc != nullptr) {
    const int pos = len - (p.query_start_loc[row + 1] - p.query_start_loc[row]);       // of the first query
    if (first + p.page_size <= first_visible(pos, p.window) && first >= p.keep_first) page = -1;
  }
  if (p.table_out != nullptr) {
    if (threadIdx.x == 0 && blockIdx.y == 0) p.table_out[(size_t)row * p.blocks + b] = page < 0 ? -1 : i * p.blocks + b;
    if (page < 0) return;             // nobody looks there
  }
  const int vectors = p.page_size * p.head_dim / 16;      // of a head
  const int live = min(max(len - first, 0), p.page_size) * p.head_dim;
  const size_t from = (size_t)max(page, 0) * p.kv_heads;
  T* out = (T*)p.out[which] + ((size_t)i * p.blocks + b) * p.kv_heads * vectors * 16;
  const uint4* in = reinterpret_cast<const uint4*>(p.pool[which]) + from * vectors;
  const int parts = gridDim.y >> 1;
#pragma unroll 4
  for (int v = part * (int)blockDim.x + threadIdx.x; v < p.kv_heads * vectors; v += parts * (int)blockDim.x) {
    const int h = v / vectors;
    const bool there = page >= 0 && (v - h * vectors) * 16 < live;
    const uint4 raw = there ? in[v] : make_uint4(0, 0, 0, 0);
    const float scale = there ? p.scale[which][from + h] : 0.f;
    const signed char* q = reinterpret_cast<const signed char*>(&raw);
#pragma unroll
    for (int e = 0; e < 16; e += Vec16<T>::N) {
      Vec16<T> x;
#pragma unroll
      for (int n = 0; n < Vec16<T>::N; ++n) x.set(n, __fmul_rn((float)q[e + n], scale));
      store16(out + (size_t)v * 16 + e, x);
    }
  }
}

}  // namespace li

using namespace li;

// The arguments of the entries of this file and its neighbours come as one structure of 8-byte fields, which the host packs in one go
// (two dozen arguments one by one cost it 4 us a call).
struct RopeKvWriteInt8Args {
  long long dtype;          // of qkv and q_out
  const void* qkv;
  long long row_stride;
  void* q_out;              // may be q's place in qkv
  long long q_out_stride;
  const int *positions, *seq_of_token, *block_table;
  long long table_stride;
  void *k_pool, *v_pool;
  float *k_scale, *v_scale;
  const float* inv_freq;    // null: nothing is rotated
  long long tokens, heads, kv_heads, head_dim, rotary_dim, page_size, num_pages;    // num_pages 0: only q is rotated
  double cs_scale;
  cudaStream_t stream;
};

// The most bytes of cosines and sines in a block of rope_kv_write_int8_kernel: what leaves an SM its blocks, and, for pages that need more, what a block
// may have.
constexpr size_t kAngleBytes = 40 * 1024, kMostAngleBytes = 200 * 1024;

template <typename T, int kWarps>
static int launch_append(const AppendParams& p, int chunk, dim3 grid, size_t shared, cudaStream_t stream) {
  static bool configured = false;
  if (shared > kAngleBytes && !configured) {
    const cudaError_t e = cudaFuncSetAttribute(rope_kv_write_int8_kernel<T, kWarps>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostAngleBytes);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  return (int)launch_pdl(p.tokens, rope_kv_write_int8_kernel<T, kWarps>, grid, dim3(kWarps * 32), shared, stream, p, chunk);
}
template <typename T>
static int launch_append_odd(const AppendParams& p, cudaStream_t stream) {
  const size_t shared = (size_t)p.page_size * (p.inv_freq != nullptr ? p.rotary_dim : 0) * sizeof(float);
  const dim3 grid(p.tokens), block(kAppendWarps * 32);
  return shared <= 48 * 1024 ? (int)launch_pdl(p.tokens, rope_kv_write_int8_odd_kernel<T, true>, grid, block, shared, stream, p)
                             : (int)launch_pdl(p.tokens, rope_kv_write_int8_odd_kernel<T, false>, grid, block, 0, stream, p);
}

// head_dim a multiple of 16, at most 512; pages of any number of tokens.
LI_EXPORT int li_rope_kv_write_int8(const RopeKvWriteInt8Args* a) {
  const int tokens = (int)a->tokens, head_dim = (int)a->head_dim;
  if (tokens == 0) return 0;
  if (a->heads < 0 || a->kv_heads < 1 || head_dim < 16 || head_dim % 16 || head_dim > 512 || a->page_size < 1 ||
      a->page_size * head_dim > 0x7fffffffL)
    return LI_ERR_UNSUPPORTED;
  if (a->inv_freq != nullptr && (a->rotary_dim < 0 || a->rotary_dim % 2 || a->rotary_dim > head_dim)) return LI_ERR_UNSUPPORTED;
  const size_t size = a->dtype == kFloat32 ? 4 : 2;
  if (!aligned16(a->qkv) || !aligned16(a->q_out) || a->row_stride * size % 16 || a->q_out_stride * size % 16 || !aligned16(a->k_pool) ||
      !aligned16(a->v_pool))
    return LI_ERR_ALIGNMENT;
  AppendParams p{a->qkv, (size_t)a->row_stride, a->q_out, (size_t)a->q_out_stride, a->positions, a->seq_of_token, a->block_table,
                 (int)a->table_stride, {(signed char*)a->k_pool, (signed char*)a->v_pool}, {a->k_scale, a->v_scale}, a->inv_freq, tokens,
                 (int)a->heads, (int)a->kv_heads, head_dim, (int)a->rotary_dim, (int)a->page_size, (int)a->num_pages, (float)a->cs_scale};
  // Few tokens are a block each (single tokens are items of their own then, and every SM gets some); the more there are, the more share
  // a block's start, its cosines and its sines, as far as these fit: a block keeps them for its own tokens and for those that end its last page.
  const size_t each = (size_t)(a->inv_freq != nullptr ? a->rotary_dim : 0) * sizeof(float), page = a->page_size;
  const size_t most = page * each <= kAngleBytes ? kAngleBytes : kMostAngleBytes;
  if (page > kMaxPage || page * each > most || each % 64) return a->dtype == kFloat32 ? launch_append_odd<float>(p, a->stream) : launch_append_odd<bf16>(p, a->stream);
  int chunk = 1;
  while (chunk < kMaxChunk && 3L * tokens > 8L * 148 * chunk) chunk *= 2;
  while (chunk > 1 && (page + chunk - 1) * each > most) chunk /= 2;
  const size_t shared = (page + chunk - 1) * each;
  const dim3 grid((tokens + chunk - 1) / chunk, a->num_pages > 0 ? 3 : 1);
  const bool few = tokens > 2048 && a->kv_heads <= 4 && a->heads * (head_dim / 16) <= 128;
  if (a->dtype == kFloat32) return few ? launch_append<float, 4>(p, chunk, grid, shared, a->stream) : launch_append<float, 8>(p, chunk, grid, shared, a->stream);
  return few ? launch_append<bf16, 4>(p, chunk, grid, shared, a->stream) : launch_append<bf16, 8>(p, chunk, grid, shared, a->stream);
}

struct ReadPagesInt8Args {
  long long dtype;          // of k_out and v_out
  const void *k_pool, *v_pool;
  const float *k_scale, *v_scale;
  const int* block_table;
  long long table_stride;
  const int* lens;
  void *k_out, *v_out;      // [rows][blocks][kv_heads][page_size][head_dim]
  long long rows, blocks, kv_heads, head_dim, page_size, num_pages;
  const int *row_index, *query_start_loc;     // these and the rest: see ReadParams
  long long window, keep_first;
  int* table_out;
  cudaStream_t stream;
};

LI_EXPORT int li_read_pages_int8(const ReadPagesInt8Args* a) {
  if (a->rows == 0 || a->blocks == 0) return 0;
  if (a->kv_heads < 1 || a->head_dim < 16 || a->head_dim % 16 || a->page_size < 1 || a->rows > 65535) return LI_ERR_UNSUPPORTED;
  if (a->kv_heads * a->page_size * a->head_dim > 0x7fffffffL) return LI_ERR_UNSUPPORTED;
  if (!aligned16(a->k_pool) || !aligned16(a->v_pool) || !aligned16(a->k_out) || !aligned16(a->v_out)) return LI_ERR_ALIGNMENT;
  ReadParams p{{(const signed char*)a->k_pool, (const signed char*)a->v_pool}, {a->k_scale, a->v_scale}, a->block_table,
               (int)a->table_stride, a->lens, a->row_index, a->query_start_loc, (int)a->window,
               a->window > 0 ? (int)a->keep_first : 0, a->table_out, {a->k_out, a->v_out}, (int)a->blocks, (int)a->kv_heads,
               (int)a->head_dim, (int)a->page_size, (int)a->num_pages};
  // A page is a block's, and of several while there are fewer of them than the device holds.
  long long parts = 1;
  while (parts < 4 && parts * 2 * 256 <= a->kv_heads * a->page_size * a->head_dim / 16 && 4 * parts * a->blocks * a->rows <= 4 * 148) parts *= 2;
  const dim3 grid((unsigned)a->blocks, 2 * (unsigned)parts, (unsigned)a->rows);
  return a->dtype == kFloat32 ? (int)launch_pdl(a->rows, read_pages_int8_kernel<float>, grid, dim3(256), 0, a->stream, p)
                              : (int)launch_pdl(a->rows, read_pages_int8_kernel<bf16>, grid, dim3(256), 0, a->stream, p);
}
