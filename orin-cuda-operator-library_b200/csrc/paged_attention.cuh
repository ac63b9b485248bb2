// Shared parts of the paged decode attention kernels: arguments, the search
// for a CTA's first tile, and where partial results lie.
#pragma once

#include <cuda_bf16.h>

#include "opl_common.cuh"
#include "paged_schedule.h"

namespace opl {

constexpr int kPagedMaxHeadDim = 256;

struct PagedArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_batch, q_head;
  int64_t k_page, k_token, k_head, v_page, v_token, v_head;
  const int* block_table;
  int64_t table_row;
  const int* seq_lens;
  int64_t pages;
  FastDiv page_size;
  int max_pages, batch, heads, kv_heads, head_dim;
  int group;          // query heads of a key-value head
  int parts;          // units a key-value head's query heads are cut into
  float scale_log2;   // score scale times log2(e)
  float* partial;     // [ctas][2][rows][head_dim], not normalised
  float2* partial_ml; // [ctas][2][rows]: maximum (log2 domain) and sum
  int* watchdog;

  __device__ __forceinline__ int units() const { return kv_heads * parts; }
};

// 2^x on the MUFU ex2 unit (relative error about 2^-22).
__device__ __forceinline__ float paged_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Loads kept after griddepcontrol.wait.
__device__ __forceinline__ int ld_int(const int* p) {
  int r;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}

__device__ __forceinline__ int paged_length(const PagedArgs& a, int sequence) {
  return readable_length(ld_int(a.seq_lens + sequence), a.max_pages,
                         static_cast<int>(a.page_size.divisor));
}

struct PagedStart {
  int64_t total;   // tiles of all units
  int64_t before;  // see segment_at
  int sequence;
  int ctas;  // that take part
};

// The whole CTA (kThreads threads) adds up the sequences' tiles and finds the
// sequence of the tile that `place(total, ctas)` names.
template <int kThreads, int kTile, int kLeast, typename Place>
__device__ __forceinline__ PagedStart paged_start(const PagedArgs& a, int grid_ctas, Place place) {
  constexpr int kWarpCount = kThreads / 32;
  __shared__ long long warp_total[kWarpCount];
  __shared__ long long found_before;
  __shared__ int found;
  const int tid = threadIdx.x;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int first = min(tid * per, a.batch), last = min(first + per, a.batch);
  long long mine = 0;
  for (int b = first; b < last; ++b) mine += key_tiles(paged_length(a, b), kTile);
  long long running = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long other = __shfl_up_sync(kFullMask, running, o);
    if ((tid & 31) >= o) running += other;
  }
  if ((tid & 31) == 31) warp_total[tid >> 5] = running;
  __syncthreads();
  long long before = running - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarpCount; ++w) {
    if (w < (tid >> 5)) before += warp_total[w];
    total += warp_total[w];
  }
  PagedStart s;
  s.total = total * a.units();
  s.ctas = active_ctas(s.total, grid_ctas, kLeast);
  const long long at = place(s.total, s.ctas);
  if (at >= 0 && at < s.total) {
    const long long wanted = at / a.units();
    if (wanted >= before && wanted < before + mine) {
      long long p = before;
      for (int b = first; b < last; ++b) {
        const int tiles = key_tiles(paged_length(a, b), kTile);
        if (wanted < p + tiles) {
          found = b;
          found_before = p;
          break;
        }
        p += tiles;
      }
    }
  }
  __syncthreads();
  s.sequence = found;
  s.before = found_before;
  return s;
}

// Rows of one unit and where its queries lie.
struct PagedUnit {
  int kv_head, first_head, rows;
};

template <int kRows>
__device__ __forceinline__ PagedUnit paged_unit(const PagedArgs& a, int unit) {
  PagedUnit u;
  u.kv_head = unit / a.parts;
  const int part = unit - u.kv_head * a.parts;
  u.first_head = u.kv_head * a.group + part * kRows;
  u.rows = min(kRows, a.group - part * kRows);
  return u;
}

// Grid and scratch of a launch: `ctas` CTAs, at most two partial units each.
struct PagedPlan {
  int rows;  // of a unit
  int ctas;
};

size_t paged_workspace_bytes(const PagedPlan& plan, int head_dim);

// The tensor-core kernel for 16-bit caches on 16-byte boundaries.
bool paged_attention_mma_supported(const PagedArgs& a, size_t element);

}  // namespace opl
