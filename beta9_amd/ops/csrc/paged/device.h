// Device helpers of the paged cache's kernels.

#pragma once

#include "paged.h"

namespace paged {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct BF16 {
  typedef __bf16 T;
};
struct FP16 {
  typedef _Float16 T;
};
struct E4M3 {
  typedef uint8_t T;
};

template <class C> struct Vec {
  typedef typename C::T x2 __attribute__((ext_vector_type(2)));
  typedef typename C::T x4 __attribute__((ext_vector_type(4)));
  typedef typename C::T x8 __attribute__((ext_vector_type(8)));
};

// A running maximum is -inf where no key has been seen, and at least kLowest where one has, also one whose score is NaN or
// -inf: a maximum passes over NaN, and what was seen must not be taken for nothing when parts are joined.
constexpr float kMinusInf = -__builtin_inff();
constexpr float kLowest = -__FLT_MAX__;

// Inclusive sums, the sum and the maximum over the lanes of whole numbers, by moves within the registers: about 50 cycles,
// where exchanges through LDS take 130 for each of the six steps.
template <int kControl, int kRows> __device__ inline int moved(int x, int otherwise) {
  return __builtin_amdgcn_update_dpp(otherwise, x, kControl, kRows, 0xf, false);
}
__device__ inline int running_sum(int x) {
  x += moved<0x111, 0xf>(x, 0);  // row_shr 1, 2, 4, 8: within 16 lanes
  x += moved<0x112, 0xf>(x, 0);
  x += moved<0x114, 0xf>(x, 0);
  x += moved<0x118, 0xf>(x, 0);
  x += moved<0x142, 0xa>(x, 0);  // the last lane of rows 0 and 2 to rows 1 and 3
  x += moved<0x143, 0xc>(x, 0);  // the last lane of the first half to the second
  return x;
}
__device__ inline int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ inline int whole_sum(int x) { return lane_value(running_sum(x), 63); }
// of values that are not negative
__device__ inline int whole_max(int x) {
  x = max(x, moved<0x111, 0xf>(x, 0));
  x = max(x, moved<0x112, 0xf>(x, 0));
  x = max(x, moved<0x114, 0xf>(x, 0));
  x = max(x, moved<0x118, 0xf>(x, 0));
  x = max(x, moved<0x142, 0xa>(x, 0));
  x = max(x, moved<0x143, 0xc>(x, 0));
  return lane_value(x, 63);
}

// Which request the packed row belongs to: the last i with cu[i] <= row, cu[requests] > row being known.
__device__ inline int request_of(const int* cu, int requests, int row) {
  int low = 0, high = requests;
  while (high - low > 1) {
    int mid = (low + high) >> 1;
    if (cu[mid] <= row)
      low = mid;
    else
      high = mid;
  }
  return low;
}

__device__ inline int clamp_int(int x, int low, int high) { return x < low ? low : (x > high ? high : x); }

// Launches a kernel of one argument block, and says whether that worked.
template <class Args> inline hipError_t launch(void (*kernel)(Args), dim3 grid, int threads, hipStream_t stream, const Args& args) {
  void* list[] = {const_cast<Args*>(&args)};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), list, 0, stream);
}

// Calls F with the types that the arguments name.
#define PAGED_DISPATCH(type, cache, F)                                                      \
  ((cache) == Type::kE4M3 ? ((type) == Type::kBF16 ? F(BF16, E4M3) : F(FP16, E4M3))         \
                          : ((type) == Type::kBF16 ? F(BF16, BF16) : F(FP16, FP16)))

// The head dim that kernels compute with: 64, 128 or 256.
inline int padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 128 ? 128 : 256); }
#define PAGED_DIM(dim, F, X, C) ((dim) <= 64 ? F(X, C, 64) : ((dim) <= 128 ? F(X, C, 128) : F(X, C, 256)))

}  // namespace paged
