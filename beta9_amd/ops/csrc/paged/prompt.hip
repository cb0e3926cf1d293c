// Causal attention of packed new tokens over their pages.
//
// o = sum_j p_j v_j / sum_j p_j over the keys that a row sees, p_j = 2^(c q.k_j - m), in one pass over the keys. The rows of
// a request and kv head are its new tokens by the G heads that share the kv head, token by token, so that a tile of 128
// rows is full for short prompts too and the keys are read once for all G. A workgroup takes one such tile, four waves 32
// rows each, and passes over the keys 64 at a time through LDS, the next 64 on their way while these are used:
//
//   S^T = K Q^T   (32x32x16) leaves lane (h, n) with row n and keys 8 (r / 4) + 4 h + r % 4, r < 16, of each 32;
//   O^T = V^T P^T wants for 16 keys eight probabilities in that lane, in any order that V shares: r = 8 u .. 8 u + 7 as
//                 they are. V's side, eight keys of one dim, is two transposing reads of LDS, of four keys each.
//
// So the probabilities never leave their registers and a row's maximum and sum are one lane's, but for one exchange between
// the two halves. Rows of LDS are 128 or 256 bytes, and the 16-byte chunks of a row are exchanged by its number so that the
// reads of eight rows' same chunk (K) and of four rows' same two chunks (V) meet no bank twice.
// LDS is one array, this kernel's own: with another beside it the compiler waits for the loads into LDS before it reads.
//
// What bounds it is the matrix instructions, the exponentials (as many cycles, nearly) and LDS (128 bytes a cycle for one
// operand of each instruction) together.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;
constexpr int kKeys = 64;

// x / d for 0 <= x < 2^31 by a product: with 2^(L - 1) < d <= 2^L, m = floor(2^(31 + L) / d) + 1 is more than 2^(31 + L) / d by
// at most 1, so x m / 2^(31 + L) exceeds x / d by less than 1 / d.
struct Divisor {
  uint32_t m, shift;
  explicit Divisor(uint32_t d = 1) {
    uint32_t log2 = 0;
    while ((1u << log2) < d) log2++;
    shift = 31 + log2;
    m = (uint32_t)((1ull << shift) / d + 1);
  }
  __device__ int divide(int x) const { return (int)((uint64_t)(uint32_t)x * m >> shift); }
};

struct PromptArgs {
  AttendArgs a;
  int q_wide;    // q's rows begin on 16 bytes
  int negative;  // the scale is below zero: q's sign is turned instead
  int group;
  Divisor by_group, by_kv_heads;
  int target_log2;  // chunks of keys wanted for all tiles of a kv head together; -1: keys are not split
  float* part;      // [items, kv heads, kRows, dim]: unnormalised sums
  float* stats;     // [items, kv heads, kRows, 2]: running maximum and sum
};

// Tiles of keys of a chunk at least.
constexpr int kLeastTiles = 4;

template <class X> struct Product;
template <> struct Product<BF16> {
  static __device__ f32x16 of(Vec<BF16>::x8 x, Vec<BF16>::x8 y, f32x16 z) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, z, 0, 0, 0); }
};
template <> struct Product<FP16> {
  static __device__ f32x16 of(Vec<FP16>::x8 x, Vec<FP16>::x8 y, f32x16 z) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, z, 0, 0, 0); }
};

template <class X> __device__ inline u32x4 widen8(u32x2 w) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if constexpr (__is_same(X, BF16)) {
      y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, false));
      y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, true));
    } else {
      y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false));
      y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true));
    }
  }
  return y;
}

// four keys of one dim: lane i of 16 gives the address of its quarter (i % 4) of row i / 4 and gets column i
__device__ inline u32x2 read_turned(const char* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// 16 bytes a lane from `from` + `at` bytes to LDS at `to` + 16 * lane. By hand, since the compiler takes a transposing read
// of LDS for one that may meet any load into LDS on its way, and would wait for the next tile there. It writes no register,
// and what it brings is read after a wait for it and a barrier. The five steps between a lane's value moved to a scalar
// register and a memory instruction that uses it are waited here too.
__device__ inline void load_into_lds(const char* from, uint32_t at, uint32_t to) {
  uint64_t address = (uint64_t)from;
  address = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(address >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)address);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(address), "s"(__builtin_amdgcn_readfirstlane(to)) : "memory", "m0");
}

template <int N> struct Constant {
  constexpr operator int() const { return N; }
};

struct Where {
  int request, tile, row0, rows, keys;  // the request's first packed row, its new tokens (as far as there are rows) and all of them
  int ahead;                            // a token's position less its number among the new ones
  int part, parts, chunk;               // of its keys, the part and its length in tiles of keys
  int index;                            // where the first of the rows' parts lies in the workspace
};

// Which rows the item stands for. The tiles that see the most keys come first, so that the last workgroups to start are
// short ones: up to 64 requests, all tiles are put in order of their last position, in 64 steps (a lane a step counts the
// tiles in it); among more, the requests follow each other, each from its last tile to its first. On 13 ragged prompts
// (16 heads of 64, up to 1500 new tokens) 71.0 us, in the requests' order 83.1.
//
// If there are few tiles, their keys are split: into chunks that are equal for all requests, as for one token. A request's
// tiles have as many parts as its last one needs; the parts of earlier tiles that hold no keys add nothing. `whole`: the item
// is a tile with all its parts (for joining them), not one part.
__device__ inline Where where_of(const PromptArgs& s, int item, bool whole) {
  const AttendArgs& a = s.a;
  int lane = threadIdx.x & 63, before = 0, items_before = 0;
  struct Request {
    int row0, until, keys, tiles;
  };
  auto request = [&](int i) {
    Request r = {0, 0, 0, 0};
    if (i < a.requests) {
      r.row0 = clamp_int(a.cu_new[i], 0, a.rows);
      r.until = max(a.cu_new[i + 1], r.row0);
      r.keys = clamp_int(a.kv_lens[i], 0, a.width << a.page_log2);
    }
    r.tiles = (int)(((int64_t)(min(r.until, a.rows) - r.row0) * s.group + kRows - 1) / kRows);
    return r;
  };
  Request mine = request(lane);
  int chunk = 0;
  if (s.target_log2 >= 0) {
    int low = 0, high = 0;
    for (int i = lane; i < a.requests; i += 64) {
      Request r = i < 64 ? mine : request(i);
      int64_t work = (int64_t)r.tiles * ((r.keys + kKeys - 1) / kKeys);
      low += (int)(work & 0xffff), high += (int)(work >> 16);  // tiles by requests are few here: see kSplitBelow
    }
    int64_t total = ((int64_t)whole_sum(high) << 16) + whole_sum(low);
    chunk = (int)min((int64_t)1 << 30, max((int64_t)kLeastTiles, (total + (1 << s.target_log2) - 1) >> s.target_log2));
  }
  for (int first = 0; first < a.requests; first += 64) {
    Request r = first ? request(first + lane) : mine;
    int from = 0, count = r.tiles, parts = 1;
    if (chunk) {
      parts = max(1, ((r.keys + kKeys - 1) / kKeys + chunk - 1) / chunk);
      count = whole ? r.tiles : r.tiles * parts;
    } else if (a.requests > 1 && a.requests <= 64) {
      // in tiles' places: the request's begin behind what it held before
      int start = (int)(min((int64_t)max(r.keys - (r.until - r.row0), 0) * s.group, (int64_t)1 << 30) / kRows), end = start + r.tiles;
      int width = (whole_max(end) + 63) / 64, low = (63 - lane) * width, here = 0;
      for (int i = 0; i < a.requests; i++)
        here += clamp_int(lane_value(end, i) - low, 0, width) - clamp_int(lane_value(start, i) - low, 0, width);
      int up = running_sum(here);
      uint64_t found = __ballot(up > item);
      if (!found) break;
      int at = __builtin_ctzll(found);
      item -= lane_value(up, at) - lane_value(here, at);
      low = (63 - at) * width;
      from = clamp_int(low - start, 0, r.tiles);
      count = clamp_int(low + width - start, 0, r.tiles) - from;
    }
    int up = running_sum(count), items_up = chunk ? running_sum(r.tiles * parts) : 0;
    uint64_t found = __ballot(before + up > item);
    if (found) {
      int at = __builtin_ctzll(found), local = item - before - lane_value(up - count, at);
      int row0 = lane_value(r.row0, at), until = lane_value(r.until, at), keys = lane_value(r.keys, at);
      Where w = {first + at, 0, row0, min(until, a.rows) - row0, keys, keys - (until - row0), 0, lane_value(parts, at), chunk, 0};
      int back = chunk && !whole ? local / w.parts : local;  // tiles from the last
      w.tile = lane_value(from + count, at) - 1 - back;
      if (chunk) {
        w.tile = lane_value(r.tiles, at) - 1 - back;
        w.part = whole ? 0 : local - back * w.parts;
        w.index = items_before + lane_value(items_up - r.tiles * parts, at) + back * w.parts;
      }
      return w;
    }
    before += lane_value(up, 63), items_before += lane_value(items_up, 63);
  }
  return {-1, 0, 0, 0, 0, 0, 0, 1, 0, 0};
}

// Waves of a SIMD, for the registers that they may have. At a head dim of 64 the pass over the keys takes 120, a narrow
// cache's more; the careful pass, in the same kernel, takes 168 and keeps some in memory for the fourth wave's sake (13 prompts
// of up to 1500 tokens, 16 heads of 64: 70.6 us with four waves, 75.0 with three; 4 of 8192: 668 and 705).
constexpr int waves_of(int dim, bool narrow) { return dim == 64 ? (narrow ? 3 : 4) : (dim == 128 ? 2 : 1); }

// D: 64, 128 or 256. A smaller head dim takes the next of these (kPad): what lies past it is zero in LDS and in q.
template <class X, class C, int D, bool kPad>
__global__ __launch_bounds__(kWaves * 64, waves_of(D, sizeof(typename C::T) == 1)) void prompt_kernel(PromptArgs s) {
  typedef typename Vec<X>::x8 Half8;
  typedef typename X::T Out;
  constexpr bool kNarrow = sizeof(typename C::T) == 1;
  constexpr float kBias = __is_same(X, FP16) ? 8.f : 0.f;   // see the kernel of one token
  constexpr float kSlack = __is_same(X, FP16) ? 6.f : 8.f;  // how far a score may pass the maximum before the sums are rescaled
  constexpr bool kAhead = D == 128;
  constexpr int kSteps = D / 16, kDims = D / 32;
  constexpr int kRowBytes = D * 2, kChunks = D / 8, kTileBytes = kKeys * kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * 2 * kTileBytes];  // [K, V][buffer][key][dim]
  const AttendArgs& a = s.a;
  const int dim = kPad ? a.dim : D;
  int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, n = lane & 31;
  int item = s.by_kv_heads.divide(blockIdx.x), kv_head = blockIdx.x - item * a.kv_heads;

  int rest = a.cu_new[a.requests], front = a.cu_new[0];  // on their way while the rest goes on
  auto clear_rest = [&]() {
    if (!a.clear_rest) return;
    rest = clamp_int(rest, 0, a.rows), front = clamp_int(front, 0, a.rows);
    for (int64_t r = blockIdx.x; r < front + (int64_t)a.rows - rest; r += gridDim.x) {
      Out* out = (Out*)a.out + (r < front ? r : r - front + rest) * a.out_row;
      for (int i = tid; i < a.heads * dim; i += kWaves * 64) out[i] = (Out)0.f;
    }
  };
  if constexpr (kPad && !kNarrow) {  // what no load writes
    for (int i = tid; i < 4 * kTileBytes / 16; i += kWaves * 64) reinterpret_cast<u32x4*>(lds)[i] = u32x4{};
    __syncthreads();
  }
  Where w = where_of(s, item, false);
  if (w.request < 0) {
    clear_rest();
    return;
  }
  int group = s.group;
  auto by_group = [&](int x) { return s.by_group.divide(x); };
  int packed = w.rows * group;  // fits: rows by heads do
  int length = w.keys;
  int ahead = w.ahead;
  int row_first = w.tile * kRows, wave_first = row_first + wave * 32;
  int row = wave_first + n;
  bool real = row < packed;
  int token = by_group(min(row, packed - 1)), head = kv_head * group + min(row, packed - 1) - token * group;
  int position = ahead + token;
  int low = ahead + by_group(min(wave_first, packed - 1)), high = ahead + by_group(min(wave_first + 31, packed - 1));
  int last = ahead + by_group(min(row_first + kRows - 1, packed - 1));  // the workgroup's last position
  int begin = w.part * w.chunk, end = last < 0 ? 0 : min(last, length - 1) / kKeys + 1;  // tiles of keys
  if (w.parts > 1) end = min(end, begin + w.chunk);

  const int* table = a.tables + w.request * a.table_stride;
  const char* caches[2] = {(const char*)a.k_cache, (const char*)a.v_cache};
  int in_page = (1 << a.page_log2) - 1;
  // the entry of the lane's key of a tile, and of the key's row of the cache
  auto entry_of = [&](int tile) { return table[min((tile * kKeys + lane) >> a.page_log2, a.width - 1)]; };
  auto cache_row = [&](int entry, int key) {
    uint32_t page = (unsigned)entry < (unsigned)a.pages ? entry : 0;
    return ((page * a.kv_heads + kv_head) << a.page_log2) + (key & in_page);  // fits: the cache has fewer than 2^32 rows
  };
  // which chunk of a key's row lies at place 0: differs for the 16 rows that a read of K covers, and by more than the pairs
  // that a read of V covers for four neighbouring rows
  auto swizzle = [](int key) { return D == 64 ? (key & 2) << 1 | (key >> 2 & 3) : (key & 3) << 2 | (key >> 2 & 3); };

  // 16-bit: straight into LDS, 1 KB an instruction, which lie in one page; the lanes fetch what belongs at their place
  constexpr int kPieceKeys = 1024 / kRowBytes, kPieces = kTileBytes / 1024 / kWaves;
  uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds) + wave * 1024;
  int piece_key = lane / kChunks;
  // a piece four further on (and twice that at a head dim of 256, where a piece is two keys) has the same exchange of chunks
  constexpr int kKinds = D == 256 ? 2 : 1;
  uint32_t piece_at[kKinds];
  bool piece_there[kKinds];
#pragma unroll
  for (int i = 0; i < kKinds; i++) {
    int chunk = (lane % kChunks) ^ swizzle((wave + kWaves * i) * kPieceKeys + piece_key);
    piece_at[i] = piece_key * dim * 2 + chunk * 16;
    piece_there[i] = !kPad || chunk * 8 < dim;
  }
  auto stage = [&](int side, int tile, int buffer, int entry) {
    uint32_t row = cache_row(entry, lane);  // the low bits of a key are its place in the tile: a tile begins on 64
    if (a.page_log2 > 6) row += (tile * kKeys) & in_page & ~(kKeys - 1);
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
      const char* from = caches[side] + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(row, (wave + kWaves * i) * kPieceKeys) * (dim * 2);
      if (piece_there[i % kKinds])
        load_into_lds(from, piece_at[i % kKinds], lds_base + (2 * side + buffer) * kTileBytes + kWaves * i * 1024);
    }
  };
  // 8-bit: through registers, widened on the way to LDS
  constexpr int kUnits = kKeys * D / 16 / (kWaves * 64);  // 16 dims each
  u32x4 narrow[kNarrow ? kUnits : 1];
  auto fetch = [&](int side, int tile, int entry) {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      int unit = tid + i * kWaves * 64, key = unit / (D / 16);
      uint64_t row = cache_row(__shfl(entry, key), tile * kKeys + key);
      int at = (unit % (D / 16)) * 16;
      const char* from = caches[side] + row * dim + at;
      if (!kPad || at + 16 <= dim) {
        narrow[i] = *reinterpret_cast<const u32x4*>(from);
      } else {
        u32x2 x = {};
        if (at + 8 <= dim) x = *reinterpret_cast<const u32x2*>(from);
        narrow[i] = u32x4{x[0], x[1], 0, 0};
      }
    }
  };
  auto put = [&](int side, int buffer) {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      int unit = tid + i * kWaves * 64, key = unit / (D / 16), chunk = (unit % (D / 16)) * 2;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        u32x2 x = {narrow[i][2 * j], narrow[i][2 * j + 1]};
        *reinterpret_cast<u32x4*>(lds + (2 * side + buffer) * kTileBytes + key * kRowBytes + ((chunk + j) ^ swizzle(key)) * 16) = widen8<X>(x);
      }
    }
  };

  Half8 q[kSteps];
  auto load_q = [&]() {
    const Out* p = (const Out*)a.q + (w.row0 + token) * a.q_row + head * a.q_head + half * 8;
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      Half8 x = {};
      if (real && (!kPad || half * 8 + 16 * i < dim)) {
        if (s.q_wide) {
          x = *reinterpret_cast<const Half8*>(p + 16 * i);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = p[16 * i + j];
        }
      }
      if (s.negative) x = -x;
      q[i] = x;
    }
  };
  f32x16 acc[kDims];
  float m, l;
  int k_at = n * kRowBytes + ((half ^ swizzle(n)) << 4);
  int quarter = lane >> 4, in_quarter = lane & 15, v_key = 4 * half + (in_quarter >> 2);
  int v_chunk = (quarter & 1) * 2 + ((in_quarter & 3) >> 1), v_rest = (in_quarter & 1) * 8;
  int v_at = v_key * kRowBytes + ((v_chunk ^ swizzle(v_key)) << 4) + v_rest;
  int v_at8 = (v_key + 8) * kRowBytes + ((v_chunk ^ swizzle(v_key + 8)) << 4) + v_rest;

  // The scores of a tile that is in LDS.
  auto scores = [&](int buffer, f32x16 (&x)[2]) {
    const char* k_lds = lds + buffer * kTileBytes;
#pragma unroll
    for (int h = 0; h < 2; h++) x[h] = f32x16{};
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        x[h] = Product<X>::of(*reinterpret_cast<const Half8*>(k_lds + h * 32 * kRowBytes + (k_at ^ (i * 32))), q[i], x[h]);
  };
  // Leaves out what a row does not see, and raises the running maximum if it must.
  auto mask = [&](f32x16 (&x)[2], int key0, uint64_t present) {
    bool whole = key0 + kKeys - 1 <= low && present == ~0ull;
    if (!whole) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        // bit 8 (r / 4) + r % 4 of a half's 32: whether the row sees the key; keys past the length lie past the position
        int count = position - key0 - 32 * h + 1;
        uint32_t seen = count <= 0 ? 0u : (count >= 32 ? ~0u : (1u << count) - 1u);
        seen = (seen & (uint32_t)(present >> (32 * h))) >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; r++) x[h][r] = seen >> (8 * (r >> 2) + (r & 3)) & 1 ? x[h][r] : kMinusInf;
      }
    }
    return whole;
  };
  auto highest = [&](const f32x16 (&x)[2]) {
    float top = kMinusInf;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 16; r++) top = fmaxf(top, x[h][r]);
    return top;
  };
  auto raise = [&](float top) {
    if (__any(top * a.score_scale > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 32)) * a.score_scale;
      top = fmaxf(m, top);
      float alpha = top == kMinusInf ? 1.f : __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kDims; d++) acc[d] *= alpha;
    }
  };
  auto weigh = [&](const f32x16 (&x)[2], Half8 (&p)[4]) {
    float from = (m == kMinusInf ? 0.f : m) - kBias;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[h][r], a.score_scale, -from));
        l += y;
        // Rounded for the matrix product; the sum l is not. The error against 64 bits is 1.25 to 1.4 times that of rounding the
        // result; what is left as a second part, as for one token, would be half as many products again.
        p[2 * h + (r >> 3)][r & 7] = (typename X::T)y;
      }
  };
  auto v_operand = [&](int buffer, int step, int d) {
    const char* v = lds + (2 + buffer) * kTileBytes + step * 16 * kRowBytes;
    u32x2 lo = read_turned(v + (v_at ^ (d * 64))), hi = read_turned(v + (v_at8 ^ (d * 64)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto values = [&](int buffer, const Half8 (&p)[4]) {
#pragma unroll
    for (int step = 0; step < 4; step++)
#pragma unroll
      for (int d = 0; d < kDims; d++) acc[d] = Product<X>::of(__builtin_bit_cast(Half8, v_operand(buffer, step, d)), p[step], acc[d]);
  };
  // The same, key by key, for the rows that see the key.
  auto values_seen = [&](int buffer, const Half8 (&p)[4], int key0, uint64_t present) {
#pragma unroll
    for (int step = 0; step < 4; step++)
#pragma unroll 1
      for (int key = 0; key < 16; key++) {
        // operand element j of half hh stands for key 8 (j / 4) + 4 hh + j % 4
        int hh = key >> 2 & 1, j = (key >> 3) * 4 + (key & 3);
        bool sees = key0 + 16 * step + key <= position && (present >> (16 * step + key) & 1);
        u32x4 only;
#pragma unroll
        for (int i = 0; i < 4; i++) only[i] = hh == half && (j >> 1) == i ? (j & 1 ? 0xffff0000u : 0xffffu) : 0u;
        u32x4 py = __builtin_bit_cast(u32x4, p[step]) & only;
#pragma unroll
        for (int d = 0; d < kDims; d++) {
          f32x16 y = Product<X>::of(__builtin_bit_cast(Half8, v_operand(buffer, step, d) & only), __builtin_bit_cast(Half8, py), acc[d]);
#pragma unroll
          for (int r = 0; r < 16; r++) acc[d][r] = sees ? y[r] : acc[d][r];
        }
      }
  };
  auto present_of = [&](int entry) { return __ballot((unsigned)entry < (unsigned)a.pages); };

  // The last loads into LDS, which nobody reads, are there before it is used for something else or given back.
  auto finish = [&]() {
    if constexpr (!kNarrow) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // One pass over the keys. A tile's scores are made in the step before its own, so that the matrix instructions of the
  // next tile's scores and the exponentials of this one's fill each other's gaps within a wave; K is therefore a tile
  // ahead of V. A later token's value that is not finite would reach the rows that do not see it through 0 * inf;
  // `careful` takes the keys of a tile one by one where a row may not see them all.
  auto pass = [&](auto careful) {
#pragma unroll
    for (int d = 0; d < kDims; d++) acc[d] = f32x16{};
    m = kMinusInf, l = 0.f;
    if (begin >= end) return;
    int mine = high < 0 ? 0 : min(end, high / kKeys + 1);  // where the wave's own tiles end
    if constexpr (!kAhead) {
      int entry0 = entry_of(begin), entry1 = entry_of(begin + 1);
      if constexpr (kNarrow) {
        fetch(0, begin, entry0), put(0, 0);
        fetch(1, begin, entry0), put(1, 0);
      } else {
        stage(0, begin, 0, entry0);
        stage(1, begin, 0, entry0);
      }
      if (!careful) load_q();
      auto step = [&](auto which, int tile) {
        constexpr int buffer = which;
        if constexpr (!kNarrow) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint64_t present = present_of(entry0);
        int entry2 = entry_of(tile + 2);
        if constexpr (kNarrow) {
          fetch(0, tile + 1, entry1);
        } else {
          stage(0, tile + 1, buffer ^ 1, entry1);
          stage(1, tile + 1, buffer ^ 1, entry1);
        }
        f32x16 x[2];
        bool whole = true;
        if (tile < mine) {
          scores(buffer, x);
          whole = mask(x, tile * kKeys, present);
          raise(highest(x));
        }
        if constexpr (kNarrow) {
          put(0, buffer ^ 1);
          fetch(1, tile + 1, entry1);
        }
        if (tile < mine) {
          Half8 p[4];
          weigh(x, p);
          if (careful && !whole)
            values_seen(buffer, p, tile * kKeys, present);
          else
            values(buffer, p);
        }
        if constexpr (kNarrow) put(1, buffer ^ 1);
        entry0 = entry1, entry1 = entry2;
      };
      for (int tile = begin; tile < end; tile += 2) {
        step(Constant<0>{}, tile);
        if (tile + 1 < end) step(Constant<1>{}, tile + 1);
      }
      finish();
      return;
    } else {
    int entry0 = entry_of(begin), entry1 = entry_of(begin + 1), entry2 = entry_of(begin + 2);  // of this tile and the next two
    if constexpr (kNarrow) {
      fetch(0, begin, entry0), put(0, 0);
      fetch(1, begin, entry0), put(1, 0);
      fetch(0, begin + 1, entry1), put(0, 1);
    } else {
      stage(0, begin, 0, entry0);
      stage(1, begin, 0, entry0);
      stage(0, begin + 1, 1, entry1);
    }
    if (!careful) load_q();
    if constexpr (!kNarrow) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    f32x16 x[2];
    scores(0, x);
    uint64_t present = present_of(entry0);
    bool whole = mask(x, begin * kKeys, present);
    raise(highest(x));
    // one step: x holds the tile's scores, y takes the next's
    auto step = [&](auto which, int tile, f32x16 (&x)[2], f32x16 (&y)[2]) {
      constexpr int buffer = which;
      constexpr bool careful_now = careful;
      if constexpr (!kNarrow) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // K of the next tile and V of this one are in LDS, and nobody reads the other buffers any more
      // the last steps load tiles that nobody uses, of the table's last entry
      int entry3 = entry_of(tile + 3);
      if constexpr (kNarrow) {
        fetch(0, tile + 2, entry2);
      } else {
        stage(0, tile + 2, buffer, entry2);
        stage(1, tile + 1, buffer ^ 1, entry1);
      }
      if (tile < mine) {
        Half8 p[4];
        scores(buffer ^ 1, y);
        weigh(x, p);
        if constexpr (kNarrow) {
          put(0, buffer);
          fetch(1, tile + 1, entry1);
        }
        if (careful && !whole)
          values_seen(buffer, p, tile * kKeys, present);
        else
          values(buffer, p);
        if constexpr (!careful_now && !kNarrow && D == 128) {
          __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
          for (int i = 0; i < 2 * kSteps; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (i < 2 * kSteps - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x2, 80 / (2 * kSteps), 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 32 / (2 * kSteps), 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
          for (int i = 0; i < 4 * kDims; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (i < 4 * kDims - 3) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          }
        }
        present = present_of(entry1);
        if (tile + 1 < mine) {
          whole = mask(y, (tile + 1) * kKeys, present);
          raise(highest(y));
        }
      } else if constexpr (kNarrow) {
        put(0, buffer);
        fetch(1, tile + 1, entry1);
      }
      if constexpr (kNarrow) put(1, buffer ^ 1);
      entry1 = entry2, entry2 = entry3;
    };
    f32x16 y[2];
    for (int tile = begin; tile < end; tile += 2) {
      step(Constant<0>{}, tile, x, y);
      if (tile + 1 < end) step(Constant<1>{}, tile + 1, y, x);
    }
    finish();
    }
  };
  pass(Constant<0>{});
  float check = 0.f;
#pragma unroll
  for (int d = 0; d < kDims; d++)
#pragma unroll
    for (int r = 0; r < 16; r++) check = __builtin_fmaf(acc[d][r], 0.f, check);
  bool again = __any(real && !(check == 0.f));
  __syncthreads();
  if (lane == 0) lds[wave] = again;
  __syncthreads();
  again = *reinterpret_cast<const uint32_t*>(lds) != 0;  // the four waves' bytes
  __syncthreads();
  if (again) pass(Constant<1>{});

  // A row that the part's first key is not too late for, and that has no maximum, saw only scores of NaN or -inf, or only
  // entries that name no page. Which of both is looked up here: in the pass it would cost registers.
  if (__any(m == kMinusInf && position >= begin * kKeys)) {
#pragma unroll 1
    for (int tile = begin; tile < end; tile++) {
      uint64_t present = present_of(entry_of(tile));
      int count = position - tile * kKeys + 1;  // keys of the tile that are not past the row
      if (count > 0 && (present << (64 - min(count, 64)))) m = fmaxf(m, kLowest);
    }
  }

  clear_rest();
  l += __shfl_xor(l, 32);
  if (w.parts > 1) {
    int64_t at = ((int64_t)(w.index + w.part) * a.kv_heads + kv_head) * kRows + wave * 32 + n;
    if (half == 0) *reinterpret_cast<f32x2*>(s.stats + 2 * at) = f32x2{m, l};
#pragma unroll
    for (int d = 0; d < kDims; d++)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<f32x4*>(s.part + at * D + 4 * half + 32 * d + 2 * r) = f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]};
    return;
  }
  float f = a.value_scale / l;  // by zero where all scores were -inf: NaN, as the formula has it
  // Through the wave's part of LDS, so that each store fills whole lines: with 16 bytes of 32 rows a store, the results of a
  // workgroup (head dim 128) took 2 us and more. Chunks are exchanged by the row as for K.
  char* mine = lds + wave * 32 * kRowBytes;
#pragma unroll
  for (int d = 0; d < kDims; d++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      typename Vec<X>::x4 y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = (Out)(m == kMinusInf ? 0.f : acc[d][r + i] * f);
      *reinterpret_cast<typename Vec<X>::x4*>(mine + n * kRowBytes + (((4 * d + r / 4) ^ (n & (kChunks - 1))) * 16) + 8 * half) = y;
    }
  int place = real ? (w.row0 + token) * a.heads + head : -1;  // fits: rows by heads do; `out` has no gaps
#pragma unroll
  for (int i = 0; i < 32 * kChunks / 64; i++) {
    int from = i * (64 / kChunks) + lane / kChunks, chunk = lane % kChunks;
    int to = __shfl(place, from);
    u32x4 y = *reinterpret_cast<const u32x4*>(mine + from * kRowBytes + chunk * 16);
    int at = (chunk ^ (from & (kChunks - 1))) * 8;
    if (to >= 0 && (!kPad || at < dim)) *reinterpret_cast<u32x4*>((Out*)a.out + (int64_t)to * dim + at) = y;
  }
}

// Joins the parts of some rows of a tile and a kv head: D / 4 threads a row, eight parts on their way at a time.
template <class X, int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs s) {
  const AttendArgs& a = s.a;
  int item = s.by_kv_heads.divide(blockIdx.x), kv_head = blockIdx.x - item * a.kv_heads;
  Where w = where_of(s, item, true);
  if (w.request < 0 || w.parts <= 1) return;
  constexpr int kLanes = D / 4, kAhead = 8;
  int dim = (threadIdx.x % kLanes) * 4, r = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes, row = w.tile * kRows + r;
  if (row >= w.rows * s.group || dim >= a.dim) return;
  float m = kMinusInf, l = 0.f;
  f32x4 o = {};
  for (int i = 0; i < w.parts; i += kAhead) {
    f32x4 x[kAhead];
    f32x2 stat[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      int64_t at = ((int64_t)(w.index + min(i + j, w.parts - 1)) * a.kv_heads + kv_head) * kRows + r;
      x[j] = *reinterpret_cast<const f32x4*>(s.part + at * D + dim);
      stat[j] = *reinterpret_cast<const f32x2*>(s.stats + 2 * at);
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (i + j >= w.parts || stat[j][0] == kMinusInf) continue;  // no key of the part is seen
      float top = fmaxf(m, stat[j][0]), f = __builtin_amdgcn_exp2f(m - top), g = __builtin_amdgcn_exp2f(stat[j][0] - top);
      l = f * l + g * stat[j][1], o = f * o + g * x[j];
      m = top;
    }
  }
  int token = s.by_group.divide(row), head = kv_head * s.group + row - token * s.group;
  typename X::T* out = (typename X::T*)a.out + (w.row0 + token) * a.out_row + head * a.out_head + dim;
  float f = a.value_scale / l;
  typename Vec<X>::x4 y;
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = (typename X::T)(m == kMinusInf ? 0.f : o[i] * f);
  *reinterpret_cast<typename Vec<X>::x4*>(out) = y;
}

int64_t tiles_of(const AttendArgs& a) { return ((int64_t)a.rows * (a.heads / a.kv_heads)) / kRows + a.requests; }

// Where fewer workgroups than this would start, and a row may see more keys than four chunks, the keys are split over about
// as many. 16 tokens behind 4096 (32 heads over 8 of 128) take 18.3 us, 70.4 without; over twice as many parts 18.7, and one
// token behind 16000 34 us instead of 26, for the joining. Among 256 tokens with nothing before them it would not pay.
constexpr int kSplitBelow = 256;
int split_log2_of(const AttendArgs& a) {
  if (tiles_of(a) * a.kv_heads >= kSplitBelow || ((int64_t)a.width << a.page_log2) <= 4 * kLeastTiles * kKeys) return -1;
  int log2 = 0;
  while ((2LL << log2) * a.kv_heads <= kSplitBelow) log2++;
  return log2;
}

}  // namespace

bool prompt_fits(const AttendArgs& a) { return (tiles_of(a) + kSplitBelow) * a.kv_heads < (1LL << 32) / (kWaves * 64); }

int64_t prompt_workspace(const AttendArgs& a) {
  int log2 = split_log2_of(a);
  return log2 < 0 ? 0 : (tiles_of(a) + (1LL << log2)) * a.kv_heads * kRows * (padded_dim(a.dim) + 2);
}

hipError_t launch_prompt(const AttendArgs& a, float* workspace, hipStream_t stream) {
  PromptArgs s;
  s.a = a;
  s.q_wide = (uintptr_t)a.q % 16 == 0 && (a.q_row | a.q_head) % 8 == 0;
  s.negative = a.score_scale < 0;
  // a scale of zero weighs all keys alike, as does one that small, and spares the kernel -inf * 0
  s.a.score_scale = a.score_scale == 0 ? 0x1p-100f : (s.negative ? -a.score_scale : a.score_scale);
  s.group = a.heads / a.kv_heads, s.by_group = Divisor(s.group), s.by_kv_heads = Divisor(a.kv_heads);
  int64_t tiles = tiles_of(a), items = tiles;
  if (items < 1) items = 1;
  s.target_log2 = split_log2_of(a);
  if (s.target_log2 >= 0) items += 1LL << s.target_log2;
  s.part = workspace, s.stats = workspace + items * a.kv_heads * kRows * padded_dim(a.dim);
  dim3 grid((unsigned)(items * a.kv_heads));
#define LAUNCH_DIM(X, C, D) (a.dim == D ? launch(prompt_kernel<X, C, D, false>, grid, kWaves * 64, stream, s) : launch(prompt_kernel<X, C, D, true>, grid, kWaves * 64, stream, s))
#define LAUNCH(X, C) PAGED_DIM(a.dim, LAUNCH_DIM, X, C)
  hipError_t status = PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
#undef LAUNCH_DIM
  if (status != hipSuccess || s.target_log2 < 0 || !tiles) return status;
  dim3 joins((unsigned)(tiles * a.kv_heads), kRows / (256 / (padded_dim(a.dim) / 4)));
#define LAUNCH_DIM(X, C, D) launch(prompt_join_kernel<X, D>, joins, 256, stream, s)
  return a.type == Type::kBF16 ? PAGED_DIM(a.dim, LAUNCH_DIM, BF16, BF16) : PAGED_DIM(a.dim, LAUNCH_DIM, FP16, FP16);
#undef LAUNCH_DIM
}

}  // namespace paged
