// The paged key-value cache on gfx950: what its kernels and their callers share.
//
// Keys and values lie as [pages, kv heads, page size, head dim], so that the page of one kv head is one contiguous
// piece of page_size * head_dim elements. tables[request][i] names the page of the request's tokens
// i * page_size .. i * page_size + page_size - 1.
//
// An entry that names no page of the cache (below 0 or past the last) is never followed: its tokens count as absent.

#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace paged {

constexpr int kMaxRequests = 4096;  // the plan's prefix sums stay in one workgroup's LDS
constexpr int kMaxHeadDim = 256;

enum class Type : int { kBF16 = 0, kFP16 = 1, kE4M3 = 2 };

struct PlanArgs {
  int* tables;  // [requests, width]
  const int* lens;
  const int* new_lens;
  const int* free_pages;  // [pages], a stack: its top lies at free_count - 1
  const int* free_count;
  int* slots;      // [tokens]
  int* positions;  // [tokens]
  int* cu_new;     // [requests + 1]
  int* kv_lens;    // [requests]
  int* lens_out;   // [requests]
  int* free_out;   // [1]
  int requests, width, pages, page_log2, tokens;
  int64_t table_stride;
};

struct ReleaseArgs {
  const int* tables;
  const int* lens;
  const uint8_t* done;
  int* free_pages;
  const int* free_count;
  int* lens_out;
  int* free_out;
  int requests, width, pages, page_log2;
  int64_t table_stride;
};

struct WriteArgs {
  const void* k;
  const void* v;
  void* k_cache;
  void* v_cache;
  const int* slots;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  int tokens, kv_heads, dim, page_log2;
  int64_t slots_in_cache;  // pages * page size
  float k_inverse, v_inverse;  // 1 / scale of an 8-bit cache
  Type type, cache;
};

struct AttendArgs {
  const void* q;
  void* out;
  const void* k_cache;
  const void* v_cache;
  const int* tables;
  const int* kv_lens;
  const int* cu_new;  // of a prompt
  int64_t q_row, q_head, out_row, out_head, table_stride;  // out has no gaps
  int rows, requests, heads, kv_heads, dim, page_log2, width, pages;
  float score_scale;  // softmax scale * scale of the keys * log2(e): exponentials are taken to the base 2
  float value_scale;
  int clear_rest;  // rows behind the last sequence: 1 clears them, 0 leaves them as they are
  Type type, cache;
};

// Each returns the launch's status.
hipError_t launch_plan(const PlanArgs& a, hipStream_t stream);
hipError_t launch_release(const ReleaseArgs& a, hipStream_t stream);
hipError_t launch_write(const WriteArgs& a, hipStream_t stream);
// workspace: as many floats as the function before says
int64_t decode_workspace(const AttendArgs& a);
hipError_t launch_decode(const AttendArgs& a, float* workspace, hipStream_t stream);
int64_t prompt_workspace(const AttendArgs& a);
bool prompt_fits(const AttendArgs& a);  // a grid's threads are counted in 32 bits
hipError_t launch_prompt(const AttendArgs& a, float* workspace, hipStream_t stream);

}  // namespace paged
