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

struct PromptArgs {
  AttendArgs a;
  int q_wide;    // q's rows begin on 16 bytes
  int negative;  // the scale is below zero: q's sign is turned instead
};

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

struct Where {
  int request, tile, row0, rows;  // the request's first packed row and its new tokens
};

// Which rows the item stands for; tiles of a request last to first, since the last see the most keys. request -1: none.
__device__ inline Where where_of(const AttendArgs& a, int item) {
  int lane = threadIdx.x & 63, group = a.heads / a.kv_heads, before = 0;
  for (int first = 0; first < a.requests; first += 64) {
    int i = first + lane, row0 = 0, n = 0;
    if (i < a.requests) {
      row0 = clamp_int(a.cu_new[i], 0, a.rows);
      n = clamp_int(a.cu_new[i + 1], row0, a.rows) - row0;
    }
    int tiles = (int)(((int64_t)n * group + kRows - 1) / kRows), up = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      int y = __shfl_up(up, d);
      if (lane >= d) up += y;
    }
    uint64_t found = __ballot(before + up > item);
    if (found) {
      int at = __builtin_ctzll(found);
      return {first + at, before + __shfl(up, at) - 1 - item, __shfl(row0, at), __shfl(n, at)};
    }
    before += __shfl(up, 63);
  }
  return {-1, 0, 0, 0};
}

template <class X, class C, int D>
__global__ __launch_bounds__(kWaves * 64, 2) void prompt_kernel(PromptArgs s) {
  typedef typename Vec<X>::x8 Half8;
  typedef typename X::T Out;
  constexpr bool kNarrow = sizeof(typename C::T) == 1;
  constexpr float kBias = __is_same(X, FP16) ? 8.f : 0.f;   // see the kernel of one token
  constexpr float kSlack = __is_same(X, FP16) ? 6.f : 8.f;  // how far a score may pass the maximum before the sums are rescaled
  constexpr int kSteps = D / 16, kDims = D / 32;
  constexpr int kRowBytes = D * 2, kChunks = D / 8, kTileBytes = kKeys * kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * 2 * kTileBytes];  // [buffer][K, V][key][dim]
  const AttendArgs& a = s.a;
  int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, n = lane & 31;
  int item = blockIdx.x / a.kv_heads, kv_head = blockIdx.x - item * a.kv_heads;

  if (a.clear_rest) {
    int rest = clamp_int(a.cu_new[a.requests], 0, a.rows), front = clamp_int(a.cu_new[0], 0, a.rows);
    for (int64_t r = blockIdx.x; r < front + (int64_t)a.rows - rest; r += gridDim.x) {
      Out* out = (Out*)a.out + (r < front ? r : r - front + rest) * a.out_row;
      for (int i = tid; i < a.heads * D; i += kWaves * 64) out[(i / D) * a.out_head + i % D] = (Out)0.f;
    }
  }
  Where w = where_of(a, item);
  if (w.request < 0) return;
  int group = a.heads / a.kv_heads;
  int packed = __builtin_amdgcn_readfirstlane(w.rows) * group;  // fits: rows by heads do
  int64_t room = (int64_t)a.width << a.page_log2;
  int length = __builtin_amdgcn_readfirstlane((int)max((int64_t)0, min((int64_t)a.kv_lens[w.request], room)));
  int ahead = length - w.rows;  // a token's position less its number among the new ones
  int row_first = __builtin_amdgcn_readfirstlane(w.tile) * kRows, wave_first = row_first + wave * 32;
  int row = wave_first + n;
  bool real = row < packed;
  int token = min(row, packed - 1) / group, head = kv_head * group + min(row, packed - 1) - token * group;
  int position = ahead + token;
  int low = ahead + min(wave_first, packed - 1) / group, high = ahead + min(wave_first + 31, packed - 1) / group;
  int last = ahead + min(row_first + kRows - 1, packed - 1) / group;  // the workgroup's last position
  int tiles = last < 0 ? 0 : min(last, length - 1) / kKeys + 1;

  Half8 q[kSteps];
  {
    const Out* p = (const Out*)a.q + (w.row0 + token) * a.q_row + head * a.q_head + half * 8;
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      Half8 x = {};
      if (real) {
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
  }

  const int* table = a.tables + w.request * a.table_stride;
  const typename C::T* caches[2] = {(const typename C::T*)a.k_cache, (const typename C::T*)a.v_cache};
  int in_page = (1 << a.page_log2) - 1;
  // the entry of the lane's key of a tile
  auto entry_of = [&](int tile) { return table[min((tile * kKeys + lane) >> a.page_log2, a.width - 1)]; };
  auto swizzle = [](int key) { return D == 128 ? (key & 7) << 1 : ((key >> 1) & 3) << 1; };

  // 16-bit: straight into LDS, 1 KB an instruction, which lie in one page; the lanes fetch what belongs at their place
  constexpr int kPieceKeys = 1024 / kRowBytes, kPieces = kTileBytes / 1024 / kWaves;
  int piece_key = lane / kChunks;
  int piece_at = piece_key * D + (((lane % kChunks) ^ swizzle(wave * kPieceKeys + piece_key)) * 8);
  auto stage = [&](int tile, int buffer, int entry) {
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
      int piece = wave + kWaves * i, key = tile * kKeys + piece * kPieceKeys;
      int page = __builtin_amdgcn_readlane(entry, piece * kPieceKeys);
      page = (unsigned)page < (unsigned)a.pages ? page : 0;
      int64_t at = ((((int64_t)page * a.kv_heads + kv_head) << a.page_log2) + (key & in_page)) * D;
#pragma unroll
      for (int side = 0; side < 2; side++)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(caches[side] + at + piece_at),
                                         (__attribute__((address_space(3))) uint32_t*)(lds + (buffer * 2 + side) * kTileBytes + piece * 1024),
                                         16, 0, 0);
    }
  };
  // 8-bit: through registers, widened on the way to LDS
  constexpr int kUnits = kKeys * D / 16 / (kWaves * 64);  // 16 dims each
  u32x4 narrow[2][kNarrow ? kUnits : 1];
  auto fetch = [&](int tile, int entry) {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      int unit = tid + i * kWaves * 64, key = unit / (D / 16), page = __shfl(entry, key);
      page = (unsigned)page < (unsigned)a.pages ? page : 0;
      int64_t at = ((((int64_t)page * a.kv_heads + kv_head) << a.page_log2) + ((tile * kKeys + key) & in_page)) * D + (unit % (D / 16)) * 16;
#pragma unroll
      for (int side = 0; side < 2; side++) narrow[side][i] = *reinterpret_cast<const u32x4*>(caches[side] + at);
    }
  };
  auto put = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      int unit = tid + i * kWaves * 64, key = unit / (D / 16), chunk = (unit % (D / 16)) * 2;
#pragma unroll
      for (int side = 0; side < 2; side++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          u32x2 x = {narrow[side][i][2 * j], narrow[side][i][2 * j + 1]};
          *reinterpret_cast<u32x4*>(lds + (buffer * 2 + side) * kTileBytes + key * kRowBytes + ((chunk + j) ^ swizzle(key)) * 16) = widen8<X>(x);
        }
    }
  };

  f32x16 acc[kDims];
  float m, l;
  int k_at = n * kRowBytes + ((half ^ swizzle(n)) << 4);
  int quarter = lane >> 4, in_quarter = lane & 15, v_key = 4 * half + (in_quarter >> 2);
  int v_at = v_key * kRowBytes + ((((quarter & 1) * 2 + ((in_quarter & 3) >> 1)) ^ swizzle(v_key)) << 4) + (in_quarter & 1) * 8;

  // One pass over the keys. A later token's value that is not finite would reach the rows that do not see it through
  // 0 * inf; `careful` takes the keys of a tile one by one where a row may not see them all.
  auto pass = [&](auto careful) {
#pragma unroll
    for (int d = 0; d < kDims; d++) acc[d] = f32x16{};
    m = kMinusInf, l = 0.f;
    if (!tiles) return;
    int entry = entry_of(0), entry_next = entry_of(1);
    if constexpr (kNarrow) {
      fetch(0, entry);
      put(0);
    } else {
      stage(0, 0, entry);
    }
    for (int tile = 0; tile < tiles; tile++) {
      int buffer = tile & 1;
      uint64_t present = __ballot((unsigned)entry < (unsigned)a.pages);
      if constexpr (!kNarrow) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // this tile is in LDS, and nobody reads the other buffer any more
      if (tile + 1 < tiles) {
        if constexpr (kNarrow)
          fetch(tile + 1, entry_next);
        else
          stage(tile + 1, buffer ^ 1, entry_next);
      }
      entry = entry_next;
      entry_next = entry_of(tile + 2);
      int key0 = tile * kKeys;
      if (key0 <= high) {
        const char* k_lds = lds + buffer * 2 * kTileBytes;
        const char* v_lds = k_lds + kTileBytes;
        f32x16 x[2] = {};
#pragma unroll
        for (int i = 0; i < kSteps; i++)
#pragma unroll
          for (int h = 0; h < 2; h++)
            x[h] = Product<X>::of(*reinterpret_cast<const Half8*>(k_lds + h * 32 * kRowBytes + (k_at ^ (i * 32))), q[i], x[h]);
        bool whole = key0 + kKeys - 1 <= low && present == ~0ull;
        // bit 8 (r / 4) + r % 4 of a half's 32: whether the row sees the key; keys past the length lie past the position
        uint32_t seen[2];
        if (!whole) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            int count = position - key0 - 32 * h + 1;
            uint32_t mask = count <= 0 ? 0u : (count >= 32 ? ~0u : (1u << count) - 1u);
            seen[h] = (mask & (uint32_t)(present >> (32 * h))) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; r++) x[h][r] = seen[h] >> (8 * (r >> 2) + (r & 3)) & 1 ? x[h][r] : kMinusInf;
          }
        }
        float top = kMinusInf;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int r = 0; r < 16; r++) top = fmaxf(top, x[h][r]);
        if (__any(top * a.score_scale > m + kSlack)) {
          top = fmaxf(top, __shfl_xor(top, 32)) * a.score_scale;
          top = fmaxf(m, top);
          float alpha = top == kMinusInf ? 1.f : __builtin_amdgcn_exp2f(m - top);
          m = top;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < kDims; d++) acc[d] *= alpha;
        }
        float from = (m == kMinusInf ? 0.f : m) - kBias;
        Half8 p[4];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            float y = __builtin_amdgcn_exp2f(__builtin_fmaf(x[h][r], a.score_scale, -from));
            l += y;
            p[2 * h + (r >> 3)][r & 7] = (typename X::T)y;  // rounded for the matrix product; the sum l is not
          }
        auto v_operand = [&](int step, int d) {
          const char* v = v_lds + step * 16 * kRowBytes + (v_at ^ (d * 64));
          u32x2 lo = read_turned(v), hi = read_turned(v + 8 * kRowBytes);
          return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        if (careful && !whole) {
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
                f32x16 y = Product<X>::of(__builtin_bit_cast(Half8, v_operand(step, d) & only), __builtin_bit_cast(Half8, py), acc[d]);
#pragma unroll
                for (int r = 0; r < 16; r++) acc[d][r] = sees ? y[r] : acc[d][r];
              }
            }
        } else {
#pragma unroll
          for (int step = 0; step < 4; step++)
#pragma unroll
            for (int d = 0; d < kDims; d++) acc[d] = Product<X>::of(__builtin_bit_cast(Half8, v_operand(step, d)), p[step], acc[d]);
        }
      }
      if constexpr (kNarrow)
        if (tile + 1 < tiles) put(buffer ^ 1);
    }
  };
  struct No { constexpr operator bool() const { return false; } };
  struct Yes { constexpr operator bool() const { return true; } };
  pass(No{});
  float check = 0.f;
#pragma unroll
  for (int d = 0; d < kDims; d++)
#pragma unroll
    for (int r = 0; r < 16; r++) check = __builtin_fmaf(acc[d][r], 0.f, check);
  if (__syncthreads_or(real && !(check == 0.f))) pass(Yes{});

  l += __shfl_xor(l, 32);
  float f = l == 0.f ? 0.f : a.value_scale / l;
  if (!real) return;
  Out* out = (Out*)a.out + (w.row0 + token) * a.out_row + head * a.out_head + 4 * half;
#pragma unroll
  for (int d = 0; d < kDims; d++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      typename Vec<X>::x4 y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = (Out)(l == 0.f ? 0.f : acc[d][r + i] * f);
      *reinterpret_cast<typename Vec<X>::x4*>(out + 32 * d + 2 * r) = y;
    }
}

}  // namespace

bool prompt_takes(const AttendArgs& a) { return a.dim == 64 || a.dim == 128; }

hipError_t launch_prompt(const AttendArgs& a, hipStream_t stream) {
  PromptArgs s;
  s.a = a;
  s.q_wide = (uintptr_t)a.q % 16 == 0 && (a.q_row | a.q_head) % 8 == 0;
  s.negative = a.score_scale < 0;
  // a scale of zero weighs all keys alike, as does one that small, and spares the kernel -inf * 0
  s.a.score_scale = a.score_scale == 0 ? 0x1p-100f : (s.negative ? -a.score_scale : a.score_scale);
  int64_t items = ((int64_t)a.rows * (a.heads / a.kv_heads)) / kRows + a.requests;
  if (items < 1) items = 1;
  if (items * a.kv_heads >= (1LL << 31)) return hipErrorInvalidValue;
  dim3 grid((unsigned)(items * a.kv_heads));
#define LAUNCH(X, C) (a.dim == 64 ? launch(prompt_kernel<X, C, 64>, grid, kWaves * 64, stream, s) : launch(prompt_kernel<X, C, 128>, grid, kWaves * 64, stream, s))
  return PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
}

}  // namespace paged
