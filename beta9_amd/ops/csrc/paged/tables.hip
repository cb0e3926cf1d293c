// Block tables and slot maps from request lengths, on the GPU: a step of a server needs no copy to the host.
//
// Request i holds l_i tokens and brings n_i: it needs ceil((l_i + n_i) / P) - ceil(l_i / P) more pages. Both the packed
// rows' beginnings and the pages' places on the free stack are prefix sums over the requests, so every workgroup
// computes them for itself (at most 4096 requests) and then writes its own
// share of the tokens and of the table rows. No workgroup waits for another, there are no atomics, and the result
// depends on nothing but the inputs. What bounds it is the launch and two dependent trips to memory.

#include <hip/hip_runtime.h>

#include "device.h"

namespace paged {
namespace {

constexpr int kThreads = 256;

// What the threads before this one hold together, and all of them, of a value that is not negative: its lower 16 bits and
// the rest are summed apart, so that 4096 values of up to 2^31 fit 32 bits. `partial`: a place in LDS of this call's own.
__device__ inline int64_t scan(int64_t x, int2* partial, int64_t& total) {
  int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int low = (int)(x & 0xffff), high = (int)(x >> 16), low_up = running_sum(low), high_up = running_sum(high);
  if (lane == 63) partial[wave] = {low_up, high_up};
  __syncthreads();
  int low_before = low_up - low, high_before = high_up - high, low_all = 0, high_all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) {
    int2 p = partial[w];
    low_before += w < wave ? p.x : 0, high_before += w < wave ? p.y : 0;
    low_all += p.x, high_all += p.y;
  }
  total = ((int64_t)high_all << 16) + low_all;
  return ((int64_t)high_before << 16) + low_before;
}

// kMost: requests that LDS has room for. (All 4096 take 64 KB: two workgroups a CU.)
template <int kMost>
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
  __shared__ int cu[kMost + 1];
  __shared__ int held[kMost];   // tokens held; -1: the request gets no slots
  __shared__ int fresh[kMost];  // its new tokens
  __shared__ int taken[kMost];  // pages taken by the requests before
  __shared__ int2 partial[3][kThreads / 64];
  int tid = threadIdx.x;
  int per = kMost == kThreads ? 1 : (a.requests + kThreads - 1) / kThreads;
  int first = tid * per, last = min(first + per, a.requests);
  int room = a.width << a.page_log2, page = 1 << a.page_log2;
  int available = clamp_int(*a.free_count, 0, a.pages);
  auto pages_of = [&](int64_t tokens) { return (int)((tokens + page - 1) >> a.page_log2); };

  int64_t sum = 0, total;
  for (int i = first; i < last; i++) {
    held[i] = clamp_int(a.lens[i], 0, room), fresh[i] = max(a.new_lens[i], 0);
    sum += fresh[i];
  }
  // a thread's 16 values of up to 2^31 pass 2^32 only where they are no lengths: their rows are past the last token then
  int64_t at = scan(min(sum, (int64_t)INT32_MAX), partial[0], total);
  int packed = (int)min(total, (int64_t)INT32_MAX);
  int need_sum = 0;
  for (int i = first; i < last; i++) {
    int64_t l = held[i], n = fresh[i];
    cu[i] = (int)min(at, (int64_t)INT32_MAX);
    at += n;
    bool fits = n > 0 && l + n <= room && at <= a.tokens;
    int need = fits ? pages_of(l + n) - pages_of(l) : 0;
    if (!fits) fresh[i] = 0;
    taken[i] = need;
    need_sum += need;
  }
  int64_t before = scan(need_sum, partial[1], total);
  int used = 0;  // this thread's, for the new top of the stack
  for (int i = first; i < last; i++) {
    int need = taken[i];
    bool granted = fresh[i] > 0 && (need == 0 || before + need <= available);
    taken[i] = (int)min(before, (int64_t)INT32_MAX);
    before += need;
    used += granted ? need : 0;
    int l = held[i], n = granted ? fresh[i] : 0;
    if (blockIdx.x == 0) {
      a.cu_new[i] = cu[i];
      a.kv_lens[i] = granted ? l + n : 0;
      a.lens_out[i] = l + n;
    }
    fresh[i] = n;
    if (!granted) held[i] = -1;
  }
  if (tid == 0) cu[a.requests] = packed;
  if (blockIdx.x == 0) {
    scan(used, partial[2], total);
    if (tid == 0) {
      a.cu_new[a.requests] = packed;
      *a.free_out = available - (int)total;
    }
  } else {
    __syncthreads();
  }

  // The new pages' entries: a wave a request. No token below reads an entry written here: those are taken from the stack.
  int lane = tid & 63, waves = gridDim.x * (kThreads / 64);
  for (int i = blockIdx.x * (kThreads / 64) + (tid >> 6); i < a.requests; i += waves) {
    if (held[i] < 0) continue;
    int have = pages_of(held[i]), want = pages_of((int64_t)held[i] + fresh[i]);
    int* row = a.tables + i * a.table_stride;
    for (int c = have + lane; c < want; c += 64) row[c] = a.free_pages[available - 1 - (taken[i] + c - have)];
  }

  for (int64_t t = (int64_t)blockIdx.x * kThreads + tid; t < a.tokens; t += (int64_t)gridDim.x * kThreads) {
    int slot = -1, position = 0;
    if (t < packed) {
      int i = request_of(cu, a.requests, (int)t);
      if (held[i] >= 0) {
        position = held[i] + (int)t - cu[i];
        int have = pages_of(held[i]), c = position >> a.page_log2;
        int p = c < have ? a.tables[i * a.table_stride + c] : a.free_pages[available - 1 - (taken[i] + c - have)];
        if ((unsigned)p < (unsigned)a.pages) slot = (p << a.page_log2) + (position & (page - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
}

__global__ __launch_bounds__(kThreads) void release_kernel(ReleaseArgs a) {
  __shared__ int2 partial[kThreads / 64];
  __shared__ int given[kMaxRequests];   // pages given back by the requests before
  __shared__ int counts[kMaxRequests];  // and by this one
  int tid = threadIdx.x;
  int per = (a.requests + kThreads - 1) / kThreads;
  int first = tid * per, last = min(first + per, a.requests);
  int room = a.width << a.page_log2, page = 1 << a.page_log2;
  int count = clamp_int(*a.free_count, 0, a.pages);
  int64_t sum = 0, total;
  for (int i = first; i < last; i++) {
    int l = clamp_int(a.lens[i], 0, room);
    bool done = a.done[i];
    counts[i] = done ? (l + page - 1) >> a.page_log2 : 0;
    sum += counts[i];
    if (blockIdx.x == 0) a.lens_out[i] = done ? 0 : l;
  }
  int64_t at = scan(min(sum, (int64_t)INT32_MAX), partial, total);
  for (int i = first; i < last; i++) {
    given[i] = (int)min(at, (int64_t)a.pages);
    at += counts[i];
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) *a.free_out = (int)min(count + total, (int64_t)a.pages);
  int lane = tid & 63, waves = gridDim.x * (kThreads / 64);
  for (int i = blockIdx.x * (kThreads / 64) + (tid >> 6); i < a.requests; i += waves) {
    for (int c = lane; c < counts[i]; c += 64) {
      int64_t place = (int64_t)count + given[i] + c;
      if (place < a.pages) a.free_pages[place] = a.tables[i * a.table_stride + c];
    }
  }
}

}  // namespace

hipError_t launch_plan(const PlanArgs& a, hipStream_t stream) {
  // a token a thread up to 1024 workgroups
  int64_t by_tokens = ((int64_t)a.tokens + kThreads - 1) / kThreads, by_rows = (a.requests + 31) / 32;
  int64_t grid = by_tokens > by_rows ? by_tokens : by_rows;
  grid = grid < 1 ? 1 : (grid > 1024 ? 1024 : grid);
  auto kernel = a.requests <= kThreads ? plan_kernel<kThreads> : (a.requests <= 1024 ? plan_kernel<1024> : plan_kernel<kMaxRequests>);
  return launch(kernel, dim3((unsigned)grid), kThreads, stream, a);
}

hipError_t launch_release(const ReleaseArgs& a, hipStream_t stream) {
  return launch(release_kernel, dim3((a.requests + 15) / 16), kThreads, stream, a);
}

}  // namespace paged
