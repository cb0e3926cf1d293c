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
  float* part;   // [items, heads, dim]: unnormalised sums
  float* stats;  // [items, heads, 2]: running maximum and sum
  int target;    // chunks wanted for all requests together; there are at most target + requests
  int least;     // keys of a chunk at least, a multiple of kWaves * kTile
  int q_wide;    // q's rows begin on 16 bytes
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
  int64_t room = (int64_t)a.width << a.page_log2;
  auto length = [&](int i) {
    int l = i < a.requests ? a.kv_lens[i] : 0;
    return (int)max((int64_t)0, min((int64_t)l, room));
  };
  int64_t total = 0;
  for (int i = lane; i < a.requests; i += 64) total += length(i);
#pragma unroll
  for (int m = 32; m; m >>= 1) total += __shfl_xor((long long)total, m);
  int64_t even = (total + s.target - 1) / s.target;
  constexpr int kStep = kWaves * kTile;
  uint32_t chunk = (uint32_t)min((int64_t)1 << 31, max((int64_t)s.least, (even + kStep - 1) / kStep * kStep));
  int before = 0;
  for (int first = 0; first < a.requests; first += 64) {
    int i = first + lane, l = length(i);
    // a request without keys has one chunk all the same: its zeros
    int n = i < a.requests ? max(1, (int)(((uint32_t)l + chunk - 1u) / chunk)) : 0;
    int up = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      int y = __shfl_up(up, d);
      if (lane >= d) up += y;
    }
    bool here = request_wanted >= 0 ? i == request_wanted : before + up > item;
    uint64_t found = __ballot(here && i < a.requests);
    if (found) {
      int at = __builtin_ctzll(found);
      int start = before + __shfl(up, at) - __shfl(n, at);
      return {first + at, __shfl(l, at), chunk, request_wanted >= 0 ? start : item - start, __shfl(n, at)};
    }
    before += __shfl(up, 63);
  }
  return {-1, 0, 0, 0, 0};
}

template <class X, class C, int D> struct Decode {
  static constexpr int kPer = D / 16;                       // dims of V a lane loads
  static constexpr bool kNarrow = sizeof(typename C::T) == 1;
  static constexpr int kLoads = kNarrow ? D / 64 : D / 32;  // 16-byte loads of a row of K a lane makes
  static constexpr int kVWords = kPer * (int)sizeof(typename C::T) / 4;
  // The exponent's offset and how far a score may pass the running maximum before the sums are rescaled. fp16 holds
  // probabilities down to 2^-24: 2^8 times larger, what is lost is below 2^-32 of the largest.
  static constexpr float kBias = __is_same(X, FP16) ? 8.f : 0.f;
  static constexpr float kSlack = __is_same(X, FP16) ? 6.f : 8.f;
  typedef typename Vec<X>::x8 Half8;

  struct Tile {
    u32x4 k[2][kLoads];
    Words<kVWords> v[8];
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

template <class X, class C, int D>
__global__ __launch_bounds__(kWaves * 64, 2) void split_kernel(SplitArgs s) {
  typedef Decode<X, C, D> K;
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
      if (c < heads_here) {
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
  const typename C::T* k_cache = (const typename C::T*)a.k_cache;
  const typename C::T* v_cache = (const typename C::T*)a.v_cache;
  int in_page = (1 << a.page_log2) - 1;
  // this lane's 8 keys: of K by its row, of V by its place; both lie on one page each
  auto entry_of = [&](int key) { return table[min(key >> a.page_log2, a.width - 1)]; };
  auto offset_of = [&](int page, int key) {
    return ((((int64_t)page * a.kv_heads + kv_head) << a.page_log2) + (key & in_page)) * D;
  };
  int k_key = 8 * (c >> 2) + (c & 3), v_key = 8 * g;
  auto fetch = [&](typename K::Tile& t, int base, int k_page, int v_page) {
    bool k_known = (unsigned)k_page < (unsigned)a.pages;
    t.known = (unsigned)v_page < (unsigned)a.pages;
    const typename C::T* k = k_cache + offset_of(k_known ? k_page : 0, base + k_key);
    const typename C::T* v = v_cache + offset_of(t.known ? v_page : 0, base + v_key) + c * K::kPer;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < K::kLoads; i++)
        t.k[h][i] = *reinterpret_cast<const u32x4*>(k + 4 * h * D + (i * 4 + g) * (16 / (int)sizeof(typename C::T)));
#pragma unroll
    for (int j = 0; j < 8; j++) t.v[j] = *reinterpret_cast<const Words<K::kVWords>*>(v + j * D);
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
        if (j >= here) t.v[j] = Words<K::kVWords>(0);  // what lies there may be no number
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
    Half8 p;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float y = __builtin_amdgcn_exp2f(x[j] - from);
      l += y;
      p[j] = (typename X::T)y;  // rounded for the matrix product; the sum l is not
    }
    // the lane's 8 keys by kPer dims, dim by dim
    uint32_t w[8][K::kPer / 2];
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
      for (int i = 0; i < K::kPer / 2; i++) {
        if constexpr (K::kNarrow)
          w[j][i] = i & 1 ? K::template widen<true>(t.v[j][i >> 1]) : K::template widen<false>(t.v[j][i >> 1]);
        else
          w[j][i] = t.v[j][i];
      }
#pragma unroll
    for (int i = 0; i < K::kPer; i++) {
      u32x4 column;
#pragma unroll
      for (int j = 0; j < 4; j++)
        column[j] = __builtin_amdgcn_perm(w[2 * j + 1][i >> 1], w[2 * j][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
      acc[i] = K::product(__builtin_bit_cast(Half8, column), p, acc[i]);
    }
  };

  // Two tiles of registers: one is computed with while the other is on its way, the entries of the table a tile ahead
  // of that.
  constexpr int kStride = kWaves * kTile;
  int base = first + wave * kTile;
  if (base < last) {
    typename K::Tile even, odd;
    fetch(even, base, entry_of(base + k_key), entry_of(base + v_key));
    int k_page = entry_of(base + kStride + k_key), v_page = entry_of(base + kStride + v_key);
    while (true) {
      bool more = base + kStride < last;
      if (more) {
        fetch(odd, base + kStride, k_page, v_page);
        k_page = entry_of(base + 2 * kStride + k_key), v_page = entry_of(base + 2 * kStride + v_key);
      }
      use(even, base);
      base += kStride;
      if (!more) break;
      more = base + kStride < last;
      if (more) {
        fetch(even, base + kStride, k_page, v_page);
        k_page = entry_of(base + 2 * kStride + k_key), v_page = entry_of(base + 2 * kStride + v_key);
      }
      use(odd, base);
      base += kStride;
      if (!more) break;
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
    float f = sum == 0.f ? 0.f : a.value_scale / sum;
#pragma unroll
    for (int i = 0; i < K::kPer; i++) out[i] = (typename X::T)(sum == 0.f ? 0.f : o[i] * f);
  } else {
    int64_t at = (int64_t)blockIdx.x * a.heads + head0 + head;
#pragma unroll
    for (int i = 0; i < K::kPer; i++) s.part[at * D + dim + i] = o[i];
    if ((threadIdx.x & 15) == 0) s.stats[2 * at] = top, s.stats[2 * at + 1] = sum;
  }
}

// Joins the chunks of one request and head: the waves take chunks in turn, a lane D / 64 dims.
template <class X, int D>
__global__ __launch_bounds__(kWaves * 64) void join_kernel(SplitArgs s) {
  const AttendArgs& a = s.a;
  __shared__ float o_lds[kWaves][D];
  __shared__ float l_lds[kWaves];
  Share share = share_of(s, 0, blockIdx.x);
  if (share.count <= 1) return;
  constexpr int kPer = D / 64;
  int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, head = blockIdx.y;
  int64_t first = share.index;
  float top = kMinusInf;
  for (int i = lane; i < share.count; i += 64) top = fmaxf(top, s.stats[2 * ((first + i) * a.heads + head)]);
  top = wave_max(top);
  float sum = 0.f, o[kPer] = {};
  for (int i = wave; i < share.count; i += kWaves) {
    int64_t at = (first + i) * a.heads + head;
    float f = top == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(s.stats[2 * at] - top);
    sum += f * s.stats[2 * at + 1];
#pragma unroll
    for (int d = 0; d < kPer; d++) o[d] += f * s.part[at * D + lane * kPer + d];
  }
#pragma unroll
  for (int d = 0; d < kPer; d++) o_lds[wave][lane * kPer + d] = o[d];
  if (lane == 0) l_lds[wave] = sum;
  __syncthreads();
  if (threadIdx.x >= D) return;
  float l = 0.f, x = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; w++) l += l_lds[w], x += o_lds[w][threadIdx.x];
  typename X::T* out = (typename X::T*)a.out + share.request * a.out_row + head * a.out_head;
  out[threadIdx.x] = (typename X::T)(l == 0.f ? 0.f : x * (a.value_scale / l));
}

constexpr int kWorkgroups = 2048;
constexpr int kLeast = 256;

int target_of(const AttendArgs& a) {
  int group = a.heads / a.kv_heads, columns = a.kv_heads * ((group + kHeads - 1) / kHeads);
  int wanted = kWorkgroups / columns;
  return wanted < 1 ? 1 : wanted;
}
// no row can have a second chunk
bool one_chunk(const AttendArgs& a) { return ((int64_t)a.width << a.page_log2) <= kLeast; }

}  // namespace

int64_t decode_workspace(const AttendArgs& a) {
  return one_chunk(a) ? 0 : ((int64_t)a.requests + target_of(a)) * a.heads * (a.dim + 2);
}

bool decode_takes(const AttendArgs& a) { return a.dim == 64 || a.dim == 128; }

hipError_t launch_decode(const AttendArgs& a, float* workspace, hipStream_t stream) {
  SplitArgs s;
  s.a = a;
  s.target = target_of(a), s.least = kLeast;
  bool single = one_chunk(a);
  int64_t items = single ? a.requests : (int64_t)a.requests + s.target;
  s.part = workspace, s.stats = workspace + items * a.heads * a.dim;
  s.q_wide = (uintptr_t)a.q % 16 == 0 && (a.q_row | a.q_head) % 8 == 0;
  int group = a.heads / a.kv_heads;
  dim3 grid((unsigned)items, (unsigned)(a.kv_heads * ((group + kHeads - 1) / kHeads)));
#define LAUNCH(X, C) \
  (a.dim == 64 ? launch(split_kernel<X, C, 64>, grid, kWaves * 64, stream, s) : launch(split_kernel<X, C, 128>, grid, kWaves * 64, stream, s))
  hipError_t status = PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
  if (status != hipSuccess || single) return status;
  dim3 rows((unsigned)a.requests, (unsigned)a.heads);
  if (a.type == Type::kBF16)
    return a.dim == 64 ? launch(join_kernel<BF16, 64>, rows, kWaves * 64, stream, s) : launch(join_kernel<BF16, 128>, rows, kWaves * 64, stream, s);
  return a.dim == 64 ? launch(join_kernel<FP16, 64>, rows, kWaves * 64, stream, s) : launch(join_kernel<FP16, 128>, rows, kWaves * 64, stream, s);
}

}  // namespace paged
