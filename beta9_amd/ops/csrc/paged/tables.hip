// Block tables and slot maps from request lengths, on the GPU: a step of a server needs no copy to the host.
//
// Request i holds l_i tokens and brings n_i: it needs ceil((l_i + n_i) / P) - ceil(l_i / P) more pages. Both the packed
// rows' beginnings and the pages' places on the free stack are prefix sums over the requests, so every workgroup
// computes them for itself (at most 4096 requests: a scan of a few microseconds out of the L2) and then writes its own
// share of the tokens and of the table rows. No workgroup waits for another, there are no atomics, and the result
// depends on nothing but the inputs. What bounds it is the launch and two dependent trips to memory.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kThreads = 256;

// Exclusive prefix sum over the workgroup of one value a thread, and the total.
__device__ inline int64_t scan(int64_t x, int64_t* partial, int64_t& total) {
  int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t up = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    int64_t y = __shfl_up((long long)up, d);
    if (lane >= d) up += y;
  }
  if (lane == 63) partial[wave] = up;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) {
    before += w < wave ? partial[w] : 0;
    total += partial[w];
  }
  __syncthreads();
  return before + up - x;
}

__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
  __shared__ int cu[kMaxRequests + 1];
  __shared__ int held[kMaxRequests];   // tokens held; -1: the request gets no slots
  __shared__ int taken[kMaxRequests];  // pages taken by the requests before
  __shared__ int64_t partial[kThreads / 64];
  int tid = threadIdx.x;
  int per = (a.requests + kThreads - 1) / kThreads;
  int first = tid * per, last = min(first + per, a.requests);
  int64_t room = (int64_t)a.width << a.page_log2;
  int page = 1 << a.page_log2;
  int available = clamp_int(*a.free_count, 0, a.pages);

  int64_t sum = 0, total;
  for (int i = first; i < last; i++) sum += max(a.new_lens[i], 0);
  int64_t at = scan(sum, partial, total);
  int packed = (int)min(total, (int64_t)INT32_MAX);
  int64_t need_sum = 0;
  for (int i = first; i < last; i++) {
    int64_t n = max(a.new_lens[i], 0);
    int64_t l = max((int64_t)0, min((int64_t)a.lens[i], room));
    cu[i] = (int)min(at, (int64_t)INT32_MAX);
    at += n;
    bool fits = n > 0 && l + n <= room && at <= a.tokens;
    int need = fits ? (int)(((l + n + page - 1) >> a.page_log2) - ((l + page - 1) >> a.page_log2)) : 0;
    held[i] = fits ? (int)l : -1;
    taken[i] = need;
    need_sum += need;
  }
  int64_t before = scan(need_sum, partial, total);
  int used = 0;  // this thread's, for the new top of the stack
  for (int i = first; i < last; i++) {
    int need = taken[i];
    bool granted = held[i] >= 0 && (need == 0 || before + need <= available);
    if (!granted) held[i] = -1;
    taken[i] = (int)min(before, (int64_t)INT32_MAX);
    before += need;
    used += granted ? need : 0;
  }
  if (tid == 0) cu[a.requests] = packed;
  __syncthreads();

  if (blockIdx.x == 0) {
    int64_t all;
    scan(used, partial, all);
    for (int i = tid; i < a.requests; i += kThreads) {
      int64_t l = max((int64_t)0, min((int64_t)a.lens[i], room));
      int n = held[i] >= 0 ? a.new_lens[i] : 0;
      a.cu_new[i] = cu[i];
      a.kv_lens[i] = held[i] >= 0 ? (int)l + n : 0;
      a.lens_out[i] = (int)l + n;
    }
    if (tid == 0) {
      a.cu_new[a.requests] = packed;
      *a.free_out = available - (int)all;
    }
  }

  // The new pages' entries: a wave a request. No token below reads an entry written here: those are taken from the stack.
  int lane = tid & 63, waves = gridDim.x * (kThreads / 64);
  for (int i = blockIdx.x * (kThreads / 64) + (tid >> 6); i < a.requests; i += waves) {
    if (held[i] < 0) continue;
    int have = (held[i] + page - 1) >> a.page_log2;
    int want = (held[i] + a.new_lens[i] + page - 1) >> a.page_log2;
    int* row = a.tables + i * a.table_stride;
    for (int c = have + lane; c < want; c += 64) row[c] = a.free_pages[available - 1 - (taken[i] + c - have)];
  }

  for (int64_t t = (int64_t)blockIdx.x * kThreads + tid; t < a.tokens; t += (int64_t)gridDim.x * kThreads) {
    int slot = -1, position = 0;
    if (t < packed) {
      int i = request_of(cu, a.requests, (int)t);
      if (held[i] >= 0) {
        position = held[i] + (int)t - cu[i];
        int have = (held[i] + page - 1) >> a.page_log2, c = position >> a.page_log2;
        int p = c < have ? a.tables[i * a.table_stride + c] : a.free_pages[available - 1 - (taken[i] + c - have)];
        if ((unsigned)p < (unsigned)a.pages) slot = (p << a.page_log2) + (position & (page - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
}

__global__ __launch_bounds__(kThreads) void release_kernel(ReleaseArgs a) {
  __shared__ int64_t partial[kThreads / 64];
  __shared__ int given[kMaxRequests];  // pages given back by the requests before
  int tid = threadIdx.x;
  int per = (a.requests + kThreads - 1) / kThreads;
  int first = tid * per, last = min(first + per, a.requests);
  int64_t room = (int64_t)a.width << a.page_log2;
  int page = 1 << a.page_log2;
  int count = clamp_int(*a.free_count, 0, a.pages);
  auto pages_of = [&](int i) {
    int64_t l = max((int64_t)0, min((int64_t)a.lens[i], room));
    return a.done[i] ? (int)((l + page - 1) >> a.page_log2) : 0;
  };
  int64_t sum = 0, total;
  for (int i = first; i < last; i++) sum += pages_of(i);
  int64_t at = scan(sum, partial, total);
  for (int i = first; i < last; i++) {
    given[i] = (int)min(at, (int64_t)a.pages);
    at += pages_of(i);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i < a.requests; i += kThreads) {
      int64_t l = max((int64_t)0, min((int64_t)a.lens[i], room));
      a.lens_out[i] = a.done[i] ? 0 : (int)l;
    }
    if (tid == 0) *a.free_out = (int)min(count + total, (int64_t)a.pages);
  }
  int lane = tid & 63, waves = gridDim.x * (kThreads / 64);
  for (int i = blockIdx.x * (kThreads / 64) + (tid >> 6); i < a.requests; i += waves) {
    int n = pages_of(i);
    for (int c = lane; c < n; c += 64) {
      int64_t place = (int64_t)count + given[i] + c;
      if (place < a.pages) a.free_pages[place] = a.tables[i * a.table_stride + c];
    }
  }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, hipStream_t stream) {
  int64_t by_tokens = (a.tokens + 4LL * kThreads - 1) / (4 * kThreads), by_rows = (a.requests + 31) / 32;
  int64_t grid = by_tokens > by_rows ? by_tokens : by_rows;
  grid = grid < 1 ? 1 : (grid > 256 ? 256 : grid);
  return launch(plan_kernel, dim3((unsigned)grid), kThreads, stream, a);
}

hipError_t launch_release(const ReleaseArgs& a, hipStream_t stream) {
  return launch(release_kernel, dim3((a.requests + 15) / 16), kThreads, stream, a);
}

}  // namespace paged
