// Attention over the paged cache, a wave for each row and head: right for every head size that is a multiple of 8 up to 256.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = c q.k_j, in one pass: a wave takes 64 keys at a time, a key
// a lane, and rescales its sums where the running maximum m rises. Everything after the loads is in 32 bits.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kWaves = 4;

template <class X, class C>
__global__ __launch_bounds__(kWaves * 64) void rows_kernel(AttendArgs a) {
  __shared__ float q_lds[kWaves][kMaxHeadDim];
  __shared__ float p_lds[kWaves][64];
  __shared__ int64_t at_lds[kWaves][64];
  int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int64_t item = (int64_t)blockIdx.x * kWaves + wave;
  bool active = item < (int64_t)a.rows * a.heads;  // the waves without an item go along to the barriers
  int row = active ? (int)(item / a.heads) : 0, head = active ? (int)(item - (int64_t)row * a.heads) : 0;
  int kv_head = head / (a.heads / a.kv_heads);
  int request = row;
  int64_t keys = 0;
  bool real = active;
  int64_t room = (int64_t)a.width << a.page_log2;
  if (active) {
    if (a.cu_new) {
      real = row < a.cu_new[a.requests] && row >= a.cu_new[0];
      if (real) {
        request = request_of(a.cu_new, a.requests, row);
        int64_t length = max((int64_t)0, min((int64_t)a.kv_lens[request], room));
        keys = min(length, max((int64_t)0, length - a.cu_new[request + 1] + row + 1));
      }
    } else {
      keys = max((int64_t)0, min((int64_t)a.kv_lens[request], room));
    }
    const typename X::T* q = (const typename X::T*)a.q + row * a.q_row + head * a.q_head;
    for (int d = lane; d < a.dim; d += 64) q_lds[wave][d] = to_float<X>(q[d]);
  }
  __syncthreads();

  float m = kMinusInf, l = 0.f, acc[kMaxHeadDim / 64] = {};
  const int* table = a.tables + request * a.table_stride;
  for (int64_t base = 0; base < keys; base += 64) {
    int64_t key = base + lane, at = -1;
    if (key < keys) {
      int page = table[key >> a.page_log2];
      if ((unsigned)page < (unsigned)a.pages)
        at = ((((int64_t)page * a.kv_heads + kv_head) << a.page_log2) + (key & ((1 << a.page_log2) - 1))) * a.dim;
    }
    float s = kMinusInf;
    if (at >= 0) {
      const typename C::T* k = (const typename C::T*)a.k_cache + at;
      s = 0.f;
      for (int d = 0; d < a.dim; d += 8) {
        float x[8];
        load8<C>(k + d, x);
#pragma unroll
        for (int i = 0; i < 8; i++) s += x[i] * q_lds[wave][d + i];
      }
      s *= a.score_scale;
    }
    float top = fmaxf(m, wave_max(s)), base_of = top == kMinusInf ? 0.f : top;
    float p = at >= 0 ? exp2f(s - base_of) : 0.f, alpha = exp2f(m - base_of);
    m = top;
    l = l * alpha + wave_sum(p);
    p_lds[wave][lane] = p;
    at_lds[wave][lane] = at;
    __builtin_amdgcn_wave_barrier();
    int count = (int)min((int64_t)64, keys - base);
#pragma unroll
    for (int j = 0; j < kMaxHeadDim / 64; j++) {
      int d = j * 64 + lane;
      if (d >= a.dim) break;
      float x = acc[j] * alpha;
      for (int i = 0; i < count; i++) {
        int64_t v_at = at_lds[wave][i];
        if (v_at >= 0) x += p_lds[wave][i] * to_float<C>(((const typename C::T*)a.v_cache)[v_at + d]);
      }
      acc[j] = x;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!active || (!real && !a.clear_rest)) return;
  typename X::T* out = (typename X::T*)a.out + row * a.out_row + head * a.out_head;
#pragma unroll
  for (int j = 0; j < kMaxHeadDim / 64; j++) {
    int d = j * 64 + lane;
    if (d < a.dim) out[d] = (typename X::T)(l == 0.f ? 0.f : acc[j] * a.value_scale / l);
  }
}

}  // namespace

hipError_t launch_attend_rows(const AttendArgs& a, hipStream_t stream) {
  int64_t items = (int64_t)a.rows * a.heads;
  if (!items) return hipSuccess;
  dim3 grid((unsigned)((items + kWaves - 1) / kWaves));
#define LAUNCH(X, C) launch(rows_kernel<X, C>, grid, kWaves * 64, stream, a)
  return PAGED_DISPATCH(a.type, a.cache, LAUNCH);
#undef LAUNCH
}

}  // namespace paged
