// New keys and values into their pages: cache[page of slot][head][slot in page] = x[token][head].
//
// A copy, bound by memory: each thread moves 8 neighbours of one row (16 bytes; 8 bytes into an 8-bit cache), so the
// threads of a token's head cover its row without gaps. An 8-bit cache holds e4m3(clamp(x / scale, +-448)): x times the
// rounded 1 / scale in 32 bits, clamped because the conversion of larger values gives NaN, NaN kept, rounded once to the
// nearest, ties to even.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kThreads = 256;

template <class X, class C, bool kWide>
__global__ __launch_bounds__(kThreads) void write_kernel(WriteArgs a) {
  int units = a.kv_heads * (a.dim / 8);
  int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  int64_t t = id / units;
  if (t >= a.tokens) return;
  int unit = (int)(id - t * units), head = unit / (a.dim / 8), d = (unit - head * (a.dim / 8)) * 8;
  int slot = a.slots[t];
  if (slot < 0 || slot >= a.slots_in_cache) return;
  int64_t to = ((((int64_t)(slot >> a.page_log2) * a.kv_heads + head) << a.page_log2) + (slot & ((1 << a.page_log2) - 1))) * a.dim + d;
#pragma unroll
  for (int side = 0; side < 2; side++) {
    const typename X::T* from = side ? (const typename X::T*)a.v + t * a.v_row + head * a.v_head + d
                                     : (const typename X::T*)a.k + t * a.k_row + head * a.k_head + d;
    typename C::T* at = (typename C::T*)(side ? a.v_cache : a.k_cache) + to;
    typename Vec<X>::x8 x;
    if (kWide) {
      x = *reinterpret_cast<const typename Vec<X>::x8*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = from[i];
    }
    if constexpr (sizeof(typename C::T) == 2) {
      *reinterpret_cast<typename Vec<X>::x8*>(at) = x;
    } else {
      float inverse = side ? a.v_inverse : a.k_inverse, y[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        y[i] = (float)x[i] * inverse;
        y[i] = y[i] > 448.f ? 448.f : (y[i] < -448.f ? -448.f : y[i]);
      }
      u32x2 packed;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
        packed[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], w, true);
      }
      *reinterpret_cast<u32x2*>(at) = packed;
    }
  }
}

}  // namespace

hipError_t launch_write(const WriteArgs& a, hipStream_t stream) {
  int64_t threads = (int64_t)a.tokens * a.kv_heads * (a.dim / 8);
  if (!threads) return hipSuccess;
  dim3 grid((unsigned)((threads + kThreads - 1) / kThreads));
  // 16-byte loads where every row begins on 16 bytes; single elements otherwise (an odd slice of a wider projection)
  bool wide = ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 && (a.k_row | a.k_head | a.v_row | a.v_head) % 8 == 0;
#define LAUNCH(X, C) (wide ? launch(write_kernel<X, C, true>, grid, kThreads, stream, a) : launch(write_kernel<X, C, false>, grid, kThreads, stream, a))
  return PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
}

}  // namespace paged
