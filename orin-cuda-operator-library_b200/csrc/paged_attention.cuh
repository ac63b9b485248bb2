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

__device__ __forceinline__ void st_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void st_out(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void st_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Joins the parts of the unit that CTA blockIdx.x of the main launch starts
// and does not end (slot 1 of that CTA, slot 0 of the following ones), row
// blockIdx.y, in key order.
template <typename T, int kUnitTile, int kUnitLeast, int kRows>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedArgs a, int grid_ctas,
                                                         int row_cap) {
  __shared__ float top_of_warp[4];
  pdl_begin();
  int64_t at = 0, limit = 0;
  const int cta = blockIdx.x;
  const PagedStart start = paged_start<128, kUnitTile, kUnitLeast>(
      a, grid_ctas, [&](long long total, int ctas) -> long long {
        if (cta + 1 >= ctas) return -1;
        limit = range_begin(total, ctas, cta + 1);
        at = limit - 1;  // the last tile of the CTA
        return at;
      });
  if (cta + 1 >= start.ctas) return;
  const int sequence = start.sequence;
  const int length = paged_length(a, sequence);
  const int tiles = key_tiles(length, kUnitTile);
  const Segment last = segment_at(at, limit, start.before, tiles, a.units());
  if (last.end == tiles) return;  // not cut here
  const int64_t unit_begin = at - last.begin;
  if (unit_begin < range_begin(start.total, start.ctas, cta)) return;  // an earlier CTA starts it
  const PagedUnit unit = paged_unit<kRows>(a, last.unit);
  const int row = blockIdx.y;
  if (row >= unit.rows) return;
  const int end_cta = range_owner(start.total, start.ctas, unit_begin + tiles - 1);
  const int parts = end_cta - cta + 1;
  const auto part_row = [&](int p) {
    const int slot = p == 0 ? 2 * cta + 1 : 2 * (cta + p);
    return static_cast<int64_t>(slot) * row_cap + row;
  };
  float top = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += 128) top = fmaxf(top, __ldcg(&a.partial_ml[part_row(p)]).x);
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) top_of_warp[threadIdx.x >> 5] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top_of_warp[0], top_of_warp[1]), fmaxf(top_of_warp[2], top_of_warp[3]));
  const float base_m = top == -INFINITY ? 0.0f : top;
  for (int d = threadIdx.x; d < a.head_dim; d += 128) {
    float sum = 0.0f, out = 0.0f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float2 ml = __ldcg(&a.partial_ml[part_row(p)]);
      const float f = paged_exp2(ml.x - base_m);
      sum = fmaf(f, ml.y, sum);
      out = fmaf(f, __ldcg(&a.partial[part_row(p) * a.head_dim + d]), out);
    }
    st_out(static_cast<T*>(a.out) +
               (static_cast<int64_t>(sequence) * a.heads + unit.first_head + row) * a.head_dim + d,
           out / sum);
  }
}

template <typename T, int kUnitTile, int kUnitLeast, int kRows>
cudaError_t launch_join(const PagedArgs& a, int grid_ctas, int row_cap, cudaStream_t stream) {
  return launch_pdl(paged_join_kernel<T, kUnitTile, kUnitLeast, kRows>,
                    dim3(grid_ctas - 1, row_cap), dim3(128), stream, a, grid_ctas, row_cap);
}

// The most CTAs of a launch; the workspace is sized for them.
inline int paged_grid_limit() { return 2 * sm_count(); }

// CTAs of a launch: at most `limit`, and no more than the longest batch that
// the block table can hold keeps busy.
inline int paged_grid(const PagedArgs& a, int limit, int tile, int least, int unit_rows) {
  const int64_t capacity = static_cast<int64_t>(a.max_pages) * a.page_size.divisor;
  const int64_t tiles = capacity <= tile ? 1 : (capacity - 1) / tile + 1;
  const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads *
                        ((a.group + unit_rows - 1) / unit_rows);
  // The product may pass 63 bits; then only its comparison with the limit counts.
  const double total = static_cast<double>(tiles) * static_cast<double>(units);
  if (total >= static_cast<double>(limit) * least) return limit;
  return active_ctas(tiles * units, limit, least);
}

// The tensor-core kernel: 16-bit types, head_dim a multiple of 8, addresses
// and strides multiples of 16 bytes.
template <typename T>
int paged_attention_mma(PagedArgs a, cudaStream_t stream);

}  // namespace opl
