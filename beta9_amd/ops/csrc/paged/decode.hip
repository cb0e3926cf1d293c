// Attention of one new token of each request over its pages: split over the cache's length, joined at the end.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = c q.k_j. Every byte of the cache is used by one workgroup
// once, with 4 G operations a value: memory bounds it, and all that matters is to keep enough loads in flight on
// enough workgroups. So a workgroup takes one kv head and one chunk of one request's keys, its four waves interleave
// tiles of 32 keys, and the matrix instructions are chosen so that nothing passes through LDS on the way:
//
//   S^T = K Q^T   (16x16x32: 16 keys by 16 heads) leaves lane (g, c) with head c and keys 8g .. 8g + 7 of the tile, since
//                 row i of the t-th product is key 8 (i / 4) + 4 t + i % 4;
//   O^T = V^T P^T (k = 32 keys) wants exactly these eight probabilities in that lane as its right operand, and on its left
//                 eight keys of one dim: lane (g, c) loads dims c D/16 .. of keys 8g .. 8g + 7, whole rows across its 16
//                 lanes, and turns its 8 x D/16 block by byte permutes.
//
// The G heads of a kv head fill the 16 columns (more than 16 take further workgroups). Chunks are equal for all requests
// and found by every workgroup from the lengths alone, so ragged batches are balanced without a schedule from the host.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;   // keys a wave takes at a time
constexpr int kHeads = 16;  // columns of a matrix instruction

template <int N> using Words = uint32_t __attribute__((ext_vector_type(N)));

struct SplitArgs {
  AttendArgs a;
  float* part;      // [items, heads, dim]: unnormalised sums
  float* stats;     // [items, heads, 2]: running maximum and sum
  int target_log2;  // chunks wanted for all requests together; there are at most as many more as requests
  int least;        // keys of a chunk at least, a multiple of kWaves * kTile
  int q_wide;       // q's rows begin on 16 bytes
};

struct Share {
  int request, keys;  // keys of the request
  uint32_t chunk;     // keys of a chunk
  int index, count;   // which of the request's chunks, of how many
};

// The chunk that item `item` stands for; request -1: none. The same in every lane.
__device__ inline Share share_of(const SplitArgs& s, int item, int request_wanted) {
  const AttendArgs& a = s.a;
  int lane = threadIdx.x & 63;
  auto length = [&](int i) { return clamp_int(i < a.requests ? a.kv_lens[i] : 0, 0, a.width << a.page_log2); };
  int mine = length(lane);  // the first 64 requests' lengths stay here for both passes
  // lengths are at most 2^30, requests 4096: the sums of their lower 16 bits and of the rest fit 32
  int low = mine & 0xffff, high = mine >> 16;
  for (int i = lane + 64; i < a.requests; i += 64) {
    int l = length(i);
    low += l & 0xffff, high += l >> 16;
  }
  int64_t total = ((int64_t)whole_sum(high) << 16) + whole_sum(low);
  int64_t even = (total + (1 << s.target_log2) - 1) >> s.target_log2;
  constexpr int kStep = kWaves * kTile;
  uint32_t chunk = (uint32_t)min((int64_t)1 << 31, max((int64_t)s.least, (even + kStep - 1) / kStep * kStep));
  int before = 0;
  for (int first = 0; first < a.requests; first += 64) {
    int i = first + lane, l = first ? length(i) : mine;
    // a request without keys has one chunk all the same: its zeros
    int n = i < a.requests ? max(1, (int)(((uint32_t)l + chunk - 1u) / chunk)) : 0;
    int up = running_sum(n);
    bool here = request_wanted >= 0 ? i == request_wanted : before + up > item;
    uint64_t found = __ballot(here && i < a.requests);
    if (found) {
      int at = __builtin_ctzll(found), count = lane_value(n, at), start = before + lane_value(up, at) - count;
      return {first + at, lane_value(l, at), chunk, request_wanted >= 0 ? start : item - start, count};
    }
    before += lane_value(up, 63);
  }
  return {-1, 0, 0, 0, 0};
}

// D: 64, 128 or 256. A smaller head dim takes the next of these (kPad): what lies past it is zero in the registers.
template <class X, class C, int D, bool kPad> struct Decode {
  static constexpr int kPer = D / 16;                       // dims of V a lane loads
  static constexpr bool kNarrow = sizeof(typename C::T) == 1;
  static constexpr int kSize = kNarrow ? 1 : 2;
  static constexpr int kLoads = kNarrow ? D / 64 : D / 32;  // 16-byte loads of a row of K a lane makes
  static constexpr int kVBytes = kPer * kSize, kVLoads = kVBytes > 16 ? kVBytes / 16 : 1, kVWords = kVBytes / kVLoads / 4;
  // The exponent's offset and how far a score may pass the running maximum before the sums are rescaled. fp16 holds
  // probabilities down to 2^-24: 2^8 times larger, what is lost is below 2^-32 of the largest.
  static constexpr float kBias = __is_same(X, FP16) ? 8.f : 0.f;
  static constexpr float kSlack = __is_same(X, FP16) ? 6.f : 8.f;
  typedef typename Vec<X>::x8 Half8;

  struct Tile {
    u32x4 k[2][kLoads];
    Words<kVWords> v[8][kVLoads];
    bool known;  // this lane's keys 8g .. 8g + 7 lie on a page
  };

  static __device__ f32x4 product(Half8 x, Half8 y, f32x4 z) {
    if constexpr (__is_same(X, BF16))
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, z, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, z, 0, 0, 0);
  }

  // two e4m3 of a word, exact in either 16-bit type
  template <bool kHigh> static __device__ uint32_t widen(uint32_t w) {
    if constexpr (__is_same(X, BF16))
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHigh));
  }

  // kBytes from `row` + `at` bytes, as far as the row's `size` goes (a multiple of 8; words of 4 bytes: of 4)
  template <int kWords> static __device__ Words<kWords> part(const char* row, int at, int size) {
    if constexpr (!kPad) return *reinterpret_cast<const Words<kWords>*>(row + at);
    Words<kWords> x = Words<kWords>(0);
    if constexpr (kWords == 4) {
      if (at + 16 <= size) {
        x = *reinterpret_cast<const Words<4>*>(row + at);
      } else if (at + 8 <= size) {
        u32x2 y = *reinterpret_cast<const u32x2*>(row + at);
        x[0] = y[0], x[1] = y[1];
      }
    } else {
      if (at + 4 * kWords <= size) x = *reinterpret_cast<const Words<kWords>*>(row + at);
    }
    return x;
  }

  // the operand of k-step s of a row of K
  static __device__ Half8 k_operand(const u32x4 (&k)[kLoads], int s) {
    if constexpr (kNarrow) {
      u32x4 x = k[s >> 1], y;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        uint32_t w = x[2 * (s & 1) + i];
        y[2 * i] = widen<false>(w), y[2 * i + 1] = widen<true>(w);
      }
      return __builtin_bit_cast(Half8, y);
    } else {
      return __builtin_bit_cast(Half8, k[s]);
    }
  }
  // where a lane's 8 dims of k-step s begin: the order of the dims is free as long as q and k share it
  static __device__ int k_dim(int s, int g) { return kNarrow ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8; }
};

template <class X, class C, int D, bool kPad>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 2 : 4) void split_kernel(SplitArgs s) {
  typedef Decode<X, C, D, kPad> K;
  typedef typename K::Half8 Half8;
  const AttendArgs& a = s.a;
  __shared__ float o_lds[kWaves][kHeads][D + 4];
  __shared__ float m_lds[kWaves][kHeads], l_lds[kWaves][kHeads];

  Share share = share_of(s, blockIdx.x, -1);
  if (share.request < 0 || share.index >= share.count) return;
  int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  int group = a.heads / a.kv_heads, head_tiles = (group + kHeads - 1) / kHeads;
  int kv_head = blockIdx.y / head_tiles, head_first = (blockIdx.y - kv_head * head_tiles) * kHeads;
  int heads_here = min(kHeads, group - head_first), head0 = kv_head * group + head_first;
  int first = (int)(share.index * share.chunk), last = (int)min((uint32_t)share.keys, first + share.chunk);

  Half8 q[D / 32];
  {
    const typename X::T* row = (const typename X::T*)a.q + share.request * a.q_row + (head0 + min(c, heads_here - 1)) * a.q_head;
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      const typename X::T* p = row + K::k_dim(i, g);
      Half8 x = {};
      if (c < heads_here && (!kPad || K::k_dim(i, g) < a.dim)) {
        if (s.q_wide) {
          x = *reinterpret_cast<const Half8*>(p);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = p[j];
        }
      }
      q[i] = x;
    }
  }

  const int* table = a.tables + share.request * a.table_stride;
  const char* k_cache = (const char*)a.k_cache;
  const char* v_cache = (const char*)a.v_cache;
  int row_bytes = (kPad ? a.dim : D) * K::kSize;
  int in_page = (1 << a.page_log2) - 1;
  // this lane's 8 keys: of K by its row, of V by its place; both lie on one page each
  auto entry_of = [&](int key) { return table[min(key >> a.page_log2, a.width - 1)]; };
  auto offset_of = [&](int page, int key) {
    return ((((int64_t)page * a.kv_heads + kv_head) << a.page_log2) + (key & in_page)) * row_bytes;
  };
  int k_key = 8 * (c >> 2) + (c & 3), v_key = 8 * g;
  auto fetch = [&](typename K::Tile& t, int base, int k_page, int v_page) {
    bool k_known = (unsigned)k_page < (unsigned)a.pages;
    t.known = (unsigned)v_page < (unsigned)a.pages;
    const char* k = k_cache + offset_of(k_known ? k_page : 0, base + k_key);
    const char* v = v_cache + offset_of(t.known ? v_page : 0, base + v_key);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < K::kLoads; i++) t.k[h][i] = K::template part<4>(k + 4 * h * row_bytes, (i * 4 + g) * 16, row_bytes);
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int i = 0; i < K::kVLoads; i++)
        t.v[j][i] = K::template part<K::kVWords>(v + j * row_bytes, c * K::kVBytes + i * 16, row_bytes);
  };

  f32x4 acc[K::kPer] = {};
  float m = kMinusInf, l = 0.f;
  auto use = [&](typename K::Tile& t, int base) {
    f32x4 score[2] = {};
#pragma unroll
    for (int i = 0; i < D / 32; i++)
#pragma unroll
      for (int h = 0; h < 2; h++) score[h] = K::product(K::k_operand(t.k[h], i), q[i], score[h]);
    float x[8], top = kMinusInf;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = score[j >> 2][j & 3] * a.score_scale;
    int here = t.known ? last - base - v_key : 0;  // how many of the lane's keys there are
    bool whole = __all(here >= 8);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[j] = j < here ? x[j] : kMinusInf;
#pragma unroll
        for (int i = 0; i < K::kVLoads; i++)
          if (j >= here) t.v[j][i] = Words<K::kVWords>(0);  // what lies there may be no number
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) top = fmaxf(top, x[j]);
    if (__any(top > m + K::kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      float alpha = top == kMinusInf ? 1.f : __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < K::kPer; i++) acc[i] *= alpha;
    }
    float from = (m == kMinusInf ? 0.f : m) - K::kBias;
    // The probabilities in two parts, what rounding to 16 bits leaves behind being the second: as exact as in 32 bits
    // for a second matrix product, which costs nothing next to the loads.
    Half8 p, rest;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float y = __builtin_amdgcn_exp2f(x[j] - from);
      l += y;
      p[j] = (typename X::T)y;
      rest[j] = (typename X::T)(y - (float)p[j]);
    }
    // the lane's 8 keys by kPer dims, dim by dim
    uint32_t w[8][K::kPer / 2];
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int i = 0; i < K::kPer / 2; i++) {
        constexpr int kEach = K::kVWords;
        if constexpr (K::kNarrow) {
          uint32_t x = t.v[j][(i >> 1) / kEach][(i >> 1) % kEach];
          w[j][i] = i & 1 ? K::template widen<true>(x) : K::template widen<false>(x);
        } else {
          w[j][i] = t.v[j][i / kEach][i % kEach];
        }
      }
    // An infinite value makes its sums infinite; a second part of zero or of another sign would make them NaN. (e4m3 has
    // no infinities.)
    bool finite = true;
    if constexpr (!K::kNarrow) {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 most = {};
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int i = 0; i < K::kPer / 2; i++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[j][i] & 0x7fff7fffu));
      finite = !__any(max(most[0], most[1]) >= (__is_same(X, BF16) ? 0x7f80 : 0x7c00));
    }
#pragma unroll
    for (int i = 0; i < K::kPer; i++) {
      u32x4 x;
#pragma unroll
      for (int j = 0; j < 4; j++)
        x[j] = __builtin_amdgcn_perm(w[2 * j + 1][i >> 1], w[2 * j][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
      acc[i] = K::product(__builtin_bit_cast(Half8, x), p, acc[i]);
      if (finite) acc[i] = K::product(__builtin_bit_cast(Half8, x), rest, acc[i]);
    }
  };

  // One tile of registers, the table's entries a tile ahead: 125 registers, so that four waves share a SIMD and one
  // computes while the others' loads are on their way. A second tile (221 registers, two waves) measured 33.4 us
  // instead of 31.6 on 32 ragged rows up to 2048, 98.9 instead of 98.5 on one of 131071 (bf16, 8 kv heads of 128).
  constexpr int kStride = kWaves * kTile;
  int base = first + wave * kTile;
  if (base < last) {
    typename K::Tile t;
    int k_page = entry_of(base + k_key), v_page = entry_of(base + v_key);
    for (; base < last; base += kStride) {
      fetch(t, base, k_page, v_page);
      k_page = entry_of(base + kStride + k_key), v_page = entry_of(base + kStride + v_key);
      use(t, base);
    }
  }

  // A head without a maximum had only scores of NaN or -inf, or no key. Which of both is looked up here: a flag kept in the
  // loop cost 0.5 percent (128 ragged rows up to 8192, e4m3).
  if (__any(m == kMinusInf)) {
    for (base = first + wave * kTile; base < last; base += kStride) {
      bool known = (unsigned)entry_of(base + v_key) < (unsigned)a.pages;
      if (__any(known && base + v_key < last)) {
        m = fmaxf(m, kLowest);
        break;
      }
    }
  }
  // the four waves' sums
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) m_lds[wave][c] = m, l_lds[wave][c] = l;
#pragma unroll
  for (int i = 0; i < K::kPer; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) o_lds[wave][c][(4 * g + r) * K::kPer + i] = acc[i][r];
  __syncthreads();
  int head = threadIdx.x >> 4, dim = (threadIdx.x & 15) * K::kPer;
  if (head >= heads_here) return;
  float top = kMinusInf, sum = 0.f, o[K::kPer] = {};
#pragma unroll
  for (int w = 0; w < kWaves; w++) top = fmaxf(top, m_lds[w][head]);
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    float f = top == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(m_lds[w][head] - top);
    sum += f * l_lds[w][head];
#pragma unroll
    for (int i = 0; i < K::kPer; i++) o[i] += f * o_lds[w][head][dim + i];
  }
  if (share.count == 1) {
    typename X::T* out = (typename X::T*)a.out + share.request * a.out_row + (head0 + head) * a.out_head + dim;
    float f = a.value_scale / sum;  // by zero where all scores were -inf: NaN, as the formula has it
#pragma unroll
    for (int i = 0; i < K::kPer; i++)
      if (!kPad || dim + i < a.dim) out[i] = (typename X::T)(top == kMinusInf ? 0.f : o[i] * f);
  } else {
    int64_t at = (int64_t)blockIdx.x * a.heads + head0 + head;
#pragma unroll
    for (int i = 0; i < K::kPer; i++) s.part[at * D + dim + i] = o[i];
    if ((threadIdx.x & 15) == 0) s.stats[2 * at] = top, s.stats[2 * at + 1] = sum;
  }
}

// Joins a request's chunks, for kJoin heads a workgroup: D / 4 threads a head, the rest of the 256 take chunks in turn,
// four on their way at a time.
template <class X, int D, int kJoin>
__global__ __launch_bounds__(kWaves * 64) void join_kernel(SplitArgs s) {
  const AttendArgs& a = s.a;
  constexpr int kLanes = D / 4, kSlots = kWaves * 64 / (kLanes * kJoin), kAhead = 4;
  __shared__ float o_lds[kSlots][kJoin][D];
  __shared__ float m_lds[kSlots][kJoin], l_lds[kSlots][kJoin];
  Share share = share_of(s, 0, blockIdx.x);
  if (share.count <= 1) return;
  int dim = (threadIdx.x % kLanes) * 4, at = threadIdx.x / kLanes, here = at % kJoin, slot = at / kJoin;
  int head = blockIdx.y * kJoin + here;
  bool real = head < a.heads;
  int64_t first = (int64_t)share.index * a.heads + (real ? head : 0);
  float m = kMinusInf, l = 0.f;
  f32x4 o = {};
  for (int i = slot; i < share.count; i += kAhead * kSlots) {
    f32x4 x[kAhead];
    f32x2 stat[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      int64_t from = first + (int64_t)min(i + j * kSlots, share.count - 1) * a.heads;
      x[j] = *reinterpret_cast<const f32x4*>(s.part + from * D + dim);
      stat[j] = *reinterpret_cast<const f32x2*>(s.stats + 2 * from);
      if (i + j * kSlots >= share.count) stat[j] = f32x2{kMinusInf, 0.f}, x[j] = f32x4{};
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < kAhead; j++) top = fmaxf(top, stat[j][0]);
    if (top == kMinusInf) continue;  // chunks without keys
    float f = __builtin_amdgcn_exp2f(m - top);
    m = top, l *= f, o *= f;
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      f = __builtin_amdgcn_exp2f(stat[j][0] - top);
      l += f * stat[j][1], o += f * x[j];
    }
  }
  *reinterpret_cast<f32x4*>(&o_lds[slot][here][dim]) = o;
  if (dim == 0) m_lds[slot][here] = m, l_lds[slot][here] = l;
  __syncthreads();
  if (slot || !real || dim >= a.dim) return;
  float top = m;
#pragma unroll
  for (int w = 1; w < kSlots; w++) top = fmaxf(top, m_lds[w][here]);
  float f = top == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(m - top);
  l *= f, o *= f;
#pragma unroll
  for (int w = 1; w < kSlots; w++) {
    f = top == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(m_lds[w][here] - top);
    l += f * l_lds[w][here], o += f * *reinterpret_cast<const f32x4*>(&o_lds[w][here][dim]);
  }
  typename X::T* out = (typename X::T*)a.out + share.request * a.out_row + head * a.out_head + dim;
  f = a.value_scale / l;
#pragma unroll
  for (int i = 0; i < 4; i++) out[i] = (typename X::T)(top == kMinusInf ? 0.f : o[i] * f);
}

// Keys of a chunk at least: shorter ones spend their time on starting and joining.
constexpr int kLeast = 256;
// Where no row can hold more keys, each is one chunk and nothing is joined: one launch instead of two. On one row of 333
// keys 5.9 us, against 5.6 + 3.8 split in two.
constexpr int kOne = 512;
// Rows of the join (requests by heads) up to which a workgroup joins one head only, with many threads along the chunks.
constexpr int kFewRows = 512;

int columns_of(const AttendArgs& a) { return a.kv_heads * ((a.heads / a.kv_heads + kHeads - 1) / kHeads); }

// Four workgroups fit a CU. One request is divided evenly, so that many chunks end together; several leave remainders,
// which finer chunks spread: 2048 workgroups took 192 us where 1024 took 215 (128 ragged rows, e4m3), and on one row of
// 131071 keys 98.5 where 1024 took 95.7.
// Powers of two, for the division in the kernel. -1: all rows are one chunk.
int target_log2_of(const AttendArgs& a) {
  int64_t room = (int64_t)a.width << a.page_log2;
  if (room <= kOne) return -1;
  int64_t wanted = (a.requests == 1 ? 1024 : 2048) / columns_of(a), most = (a.requests * room + kLeast - 1) / kLeast;
  int log2 = 0;
  while ((2LL << log2) <= wanted && (1LL << log2) < most) log2++;
  return log2;
}
int64_t items_of(const AttendArgs& a) {
  int log2 = target_log2_of(a);
  return (int64_t)a.requests + (log2 < 0 ? 0 : 1LL << log2);
}

}  // namespace

int64_t decode_workspace(const AttendArgs& a) {
  return target_log2_of(a) < 0 ? 0 : items_of(a) * a.heads * (padded_dim(a.dim) + 2);
}

hipError_t launch_decode(const AttendArgs& a, float* workspace, hipStream_t stream) {
  SplitArgs s;
  s.a = a;
  int log2 = target_log2_of(a);
  bool split = log2 >= 0;
  // not split: chunks of kOne, whatever the sum of the lengths is
  s.target_log2 = split ? log2 : 30, s.least = split ? kLeast : kOne;
  int64_t items = items_of(a);
  s.part = workspace, s.stats = workspace + items * a.heads * padded_dim(a.dim);
  s.q_wide = (uintptr_t)a.q % 16 == 0 && (a.q_row | a.q_head) % 8 == 0;
  dim3 grid((unsigned)items, (unsigned)columns_of(a));
#define LAUNCH_DIM(X, C, D) (a.dim == D ? launch(split_kernel<X, C, D, false>, grid, kWaves * 64, stream, s) : launch(split_kernel<X, C, D, true>, grid, kWaves * 64, stream, s))
#define LAUNCH(X, C) PAGED_DIM(a.dim, LAUNCH_DIM, X, C)
  hipError_t status = PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
#undef LAUNCH_DIM
  if (status != hipSuccess || !split) return status;
  bool few = (int64_t)a.requests * a.heads <= kFewRows;
  int join = few ? 1 : (a.dim > 128 ? 4 : 8);
  dim3 rows((unsigned)a.requests, (unsigned)((a.heads + join - 1) / join));
#define LAUNCH_DIM(X, C, D) (few ? launch(join_kernel<X, D, 1>, rows, kWaves * 64, stream, s) : launch(join_kernel<X, D, D == 256 ? 4 : 8>, rows, kWaves * 64, stream, s))
  return a.type == Type::kBF16 ? PAGED_DIM(a.dim, LAUNCH_DIM, BF16, BF16) : PAGED_DIM(a.dim, LAUNCH_DIM, FP16, FP16);
#undef LAUNCH_DIM
}

}  // namespace paged
