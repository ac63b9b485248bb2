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
  FastDiv parts;      // units a key-value head's query heads are cut into
  FastDiv units;      // of a sequence: key-value heads times parts
  float scale_log2;   // score scale times log2(e)
  int row_cap;         // the most rows of a unit, min(group, the kernel's)
  float* partial;      // [ctas][2][row_cap][head_dim], not normalised
  float2* partial_ml;  // [ctas][2][row_cap]: maximum (log2 domain) and sum
  float* aside;        // parts put aside that shared memory has no room for
  int* watchdog;
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

// The same from L2: for a launch that may share its SM's L1 with an earlier one.
__device__ __forceinline__ int ld_int_l2(const int* p) {
  int r;
  asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}

__device__ __forceinline__ int readable(const PagedArgs& a, int raw_length) {
  return readable_length(raw_length, a.max_pages, static_cast<int>(a.page_size.divisor));
}

struct PagedTotal {
  int64_t tiles;  // of all units
  int ctas;       // that take part
  Ranges ranges;  // of their warps
};

// The sequence of a tile.
struct PagedStart {
  int sequence, length, raw_length;  // as read, and as given
  int64_t before;                    // see place_of
};

__device__ __forceinline__ uint32_t warp_prefix(uint32_t x, int lane) {  // with x itself
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t other = __shfl_up_sync(kFullMask, x, o);
    if (lane >= o) x += other;
  }
  return x;
}

// A warp adds up the sequences' tiles and finds the sequence of the tile
// place(total) (none when that is negative).  Every warp does it for itself:
// this is the start of the launch, where a barrier and what it orders would
// cost more than the repeated loads.  kUnitWarps: warps of a CTA of the main
// launch.  The sums fit 32 bits (see the limit on the cache's capacity).
template <int kTile, int kUnitWarps, bool kFromL2, typename Place>
__device__ __forceinline__ PagedTotal paged_start(const PagedArgs& a, int grid_ctas,
                                                  PagedStart* start, Place place) {
  const int lane = threadIdx.x & 31;
  const auto raw_of = [&](int b) {
    return kFromL2 ? ld_int_l2(a.seq_lens + b) : ld_int(a.seq_lens + b);
  };
  const auto tiles_of = [&](int b) -> uint32_t { return key_tiles(readable(a, raw_of(b)), kTile); };
  // Lane x adds up the tiles of `per` sequences: its own loads up to 512
  // sequences, beyond that (1024: 68 against 74 us for the call) sums of 32 that
  // the warp loads together.
  uint32_t mine = 0;
  int per = (a.batch + 31) / 32, raw = 0;
  if (per == 1) {
    if (lane < a.batch) {
      raw = raw_of(lane);
      mine = key_tiles(readable(a, raw), kTile);
    }
  } else if (per <= 16) {
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
      const int b = lane * per + i;
      if (b < a.batch) mine += tiles_of(b);
    }
  } else {
    per = 32 * ((per + 31) / 32);
    int adder = 0, left = per;
#pragma unroll 8
    for (int b = lane; b - lane < a.batch; b += 32) {
      const uint32_t sum = __reduce_add_sync(kFullMask, b < a.batch ? tiles_of(b) : 0u);
      if (lane == adder) mine += sum;
      if ((left -= 32) == 0) left = per, ++adder;
    }
  }
  const uint32_t end = warp_prefix(mine, lane);
  PagedTotal total;
  total.tiles = static_cast<int64_t>(__shfl_sync(kFullMask, end, 31)) * a.units.divisor;
  total.ctas = active_ctas(total.tiles, grid_ctas, kUnitWarps);  // a tile for each warp
  total.ranges = make_ranges(total.tiles, kUnitWarps * total.ctas);
  const int64_t at = place(total);
  if (at < 0) return total;
  const uint32_t wanted =
      at >> 31 == 0 ? fast_div(static_cast<uint32_t>(at), a.units)
                    : static_cast<uint32_t>(at / a.units.divisor);
  // The lane whose sequences hold it, then the sequence among them.
  const int owner = __popc(__ballot_sync(kFullMask, end <= wanted));
  uint32_t before = __shfl_sync(kFullMask, end - mine, owner);
  if (per == 1) {
    start->sequence = owner;
    start->raw_length = __shfl_sync(kFullMask, raw, owner);
    start->length = readable(a, start->raw_length);
    start->before = before;
    return total;
  }
  for (int i = 0; i < per; i += 32) {
    const int b = owner * per + i + lane;
    const bool there = i + lane < per && b < a.batch;
    raw = there ? raw_of(b) : 0;
    const int length = readable(a, raw);
    const uint32_t tiles = there ? key_tiles(length, kTile) : 0;
    const uint32_t upto = before + warp_prefix(tiles, lane);
    const uint32_t passed = __ballot_sync(kFullMask, upto <= wanted);
    if (passed != kFullMask) {
      const int which = __popc(passed);
      start->sequence = owner * per + i + which;
      start->length = __shfl_sync(kFullMask, length, which);
      start->raw_length = __shfl_sync(kFullMask, raw, which);
      start->before = __shfl_sync(kFullMask, upto - tiles, which);
      break;
    }
    before = __shfl_sync(kFullMask, upto, 31);
  }
  return total;
}

// Rows of one unit and where its queries lie.
struct PagedUnit {
  int kv_head, first_head, rows;
};

template <int kRows>
__device__ __forceinline__ PagedUnit paged_unit(const PagedArgs& a, int unit) {
  PagedUnit u;
  u.kv_head = static_cast<int>(fast_div(unit, a.parts));
  const int part = unit - u.kv_head * static_cast<int>(a.parts.divisor);
  u.first_head = u.kv_head * a.group + part * kRows;
  u.rows = min(kRows, a.group - part * kRows);
  return u;
}

__device__ __forceinline__ void st_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void st_out(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void st_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Stores kWidth consecutive elements.
template <int kWidth, typename T>
__device__ __forceinline__ void st_row(T* p, const float (&x)[kWidth]) {
  if constexpr (kWidth == 1) {
    st_out(p, x[0]);
  } else {
    static_assert(kWidth == 4, "one or four");
    alignas(4 * sizeof(T)) T y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) st_out(&y[i], x[i]);
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(y);
    else
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(y);
  }
}

// kWidth consecutive floats that this CTA has written.
template <int kWidth>
__device__ __forceinline__ void ld_row(const float* p, float (&x)[kWidth]) {
  if constexpr (kWidth == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    x[0] = *p;
  }
}

// The same written by another launch.
template <int kWidth>
__device__ __forceinline__ void ld_row_l2(const float* p, float (&x)[kWidth]) {
  if constexpr (kWidth == 4) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    x[0] = __ldcg(p);
  }
}

// The least maximum of a part.  A part without keys (of pages outside the cache)
// has -infinity, and where all parts of a unit have, the result is zero.  One
// whose keys all score -infinity has the lowest number, so that nothing but such
// parts gives 0 / 0, as the formula does.
__device__ __forceinline__ float least_maximum(bool keys) {
  return keys ? -3.402823466e38f : -INFINITY;
}

// Whether any of a sequence's keys first .. end - 1 lies in the cache.
__device__ __forceinline__ bool any_page(const PagedArgs& a, int sequence, int first, int end) {
  bool found = false;
#pragma unroll 1
  for (int key = first + (threadIdx.x & 31); key < end && !found; key += 32)
    found = cache_page(ld_int(a.block_table + sequence * a.table_row + fast_div(key, a.page_size)),
                       a.pages);
  return __any_sync(kFullMask, found);
}

// What the warps of a CTA leave for one another in shared memory.
template <int kWarps, int kRows>
struct PagedParts {
  PartRecord records[kWarps][2];
  float m[kWarps][2][kRows], l[kWarps][2][kRows];  // log2 domain; sums
  float weight[kWarps][2][kRows];                  // of the part in its unit
  float top[kWarps][2][kRows], sum[kWarps][2][kRows];  // of the unit
};

// Joins the parts that the CTA's warps left, after a __syncthreads, and writes
// each unit to the output or, when it reaches past the CTA, to the CTA's
// partial slots.  The parts' rows, kPitch floats each, lie at rows + warp *
// kStride, or at heads + warp * kRows * kPitch when put aside.
template <typename T, int kWarps, int kRows, int kStride, int kPitch, int kWidth>
__device__ __forceinline__ void paged_merge(const PagedArgs& a, PagedParts<kWarps, kRows>& parts,
                                            const float* rows, const float* heads) {
  static_assert(kWarps <= 16, "a lane for each part");
  const int lane = threadIdx.x & 31;
  bool present = false, starts = false;
  if (lane < 2 * kWarps) {
    const PartRecord& r = parts.records[lane >> 1][lane & 1];
    present = !r.empty();
    starts = starts_unit(r, lane & 1);
  }
  const uint32_t all = __ballot_sync(kFullMask, present);
  const uint32_t first = __ballot_sync(kFullMask, starts);
  // A thread for each part and row: the part's weight in its unit.
  const auto start_of = [&](int part) {  // the first part of the unit
    return 31 - __clz(first & ((2u << part) - 1));
  };
  for (int i = threadIdx.x; i < 2 * kWarps * a.row_cap; i += 32 * kWarps) {
    const int part = i % (2 * kWarps), row = i / (2 * kWarps);
    if ((all >> part & 1u) == 0) continue;
    const uint32_t mine = parts_of_unit(all, first, start_of(part));
    float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
    for (int b = 0; b < kWarps; ++b) {  // a warp has at most one part of a unit
      const uint32_t kinds = mine >> (2 * b) & 3u;
      if (kinds != 0) top = fmaxf(top, parts.m[b][kinds >> 1][row]);
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
    for (int b = 0; b < kWarps; ++b) {
      const uint32_t kinds = mine >> (2 * b) & 3u;
      if (kinds != 0)
        sum = fmaf(paged_exp2(parts.m[b][kinds >> 1][row] - base), parts.l[b][kinds >> 1][row], sum);
    }
    parts.weight[part >> 1][part & 1][row] =
        paged_exp2(parts.m[part >> 1][part & 1][row] - base);
    parts.top[part >> 1][part & 1][row] = top;
    parts.sum[part >> 1][part & 1][row] = sum;
  }
  __syncthreads();
  const int pieces = a.head_dim / kWidth, warp = threadIdx.x >> 5;
  // A few units: the warps share the rows of each.  Many, of short sequences: a
  // warp each.
  const bool together = __popc(first) <= 2;
  constexpr int kAtOnce = 4;  // rows whose loads do not wait for one another
  int turn = 0;
  for (uint32_t left = first; left != 0; left &= left - 1, ++turn) {
    if (!together && turn % kWarps != warp) continue;
    const int start = __ffs(left) - 1;
    const uint32_t mine = parts_of_unit(all, first, start);
    const int last = 31 - __clz(mine);
    const PartRecord& r = parts.records[start >> 1][start & 1];
    const bool whole = r.begin == 0 && parts.records[last >> 1][last & 1].end == r.tiles;
    const PagedUnit unit = paged_unit<kRows>(a, r.unit);
    const int step = together ? kWarps : 1;
    for (int row = together ? warp : 0; row < unit.rows; row += kAtOnce * step) {
      for (int d = lane * kWidth; d < pieces * kWidth; d += 32 * kWidth) {
        float out[kAtOnce][kWidth] = {};
#pragma unroll 2
        for (int b = 0; b < kWarps; ++b) {
          const uint32_t kinds = mine >> (2 * b) & 3u;
          if (kinds == 0) continue;
          const int kind = kinds >> 1;
          const float* const src = parts.records[b][kind].aside != 0 ? heads + b * kRows * kPitch
                                                                     : rows + b * kStride;
          float v[kAtOnce][kWidth];
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q)
            if (row + q * step < unit.rows) ld_row(src + (row + q * step) * kPitch + d, v[q]);
#pragma unroll
          for (int q = 0; q < kAtOnce; ++q) {
            if (row + q * step >= unit.rows) continue;
            const float f = parts.weight[b][kind][row + q * step];
#pragma unroll
            for (int e = 0; e < kWidth; ++e) out[q][e] = fmaf(f, v[q][e], out[q][e]);
          }
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const int at = row + q * step;
          if (at >= unit.rows) continue;
          const float sum = parts.sum[start >> 1][start & 1][at];
          const bool none = parts.top[start >> 1][start & 1][at] == -INFINITY;  // no key
          if (whole) {
#pragma unroll
            for (int e = 0; e < kWidth; ++e)
              out[q][e] = none ? 0.0f : __fdividef(out[q][e], sum);
            st_row(static_cast<T*>(a.out) +
                       (static_cast<int64_t>(r.sequence) * a.heads + unit.first_head + at) * a.head_dim +
                       d,
                   out[q]);
          } else {
            const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (r.begin == 0 ? 1 : 0);
            st_row(a.partial + (slot * a.row_cap + at) * a.head_dim + d, out[q]);
            if (d == 0)
              a.partial_ml[slot * a.row_cap + at] =
                  make_float2(parts.top[start >> 1][start & 1][at], sum);
          }
        }
      }
    }
  }
}

// Joins the parts of the unit that CTA blockIdx.x of the main launch starts
// and does not end (slot 1 of that CTA, slot 0 of the following ones), row
// blockIdx.y, in key order: warp w takes parts w, w + 8, ...
constexpr int kJoinThreads = 256;

template <typename T, int kUnitTile, int kUnitWarps, int kRows, int kWidth>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a, int grid_ctas) {
  constexpr int kJoinWarps = kJoinThreads / 32;
  constexpr int kHeld = kPagedMaxHeadDim / (32 * kWidth);  // pieces of a lane
  __shared__ float warp_top[kJoinWarps], warp_sum[kJoinWarps];
  __shared__ float rows[kJoinWarps][kPagedMaxHeadDim];
  __shared__ int found_sequence, found_unit, found_parts;
  const int cta = blockIdx.x, row = blockIdx.y;
  // The main launch waits for everything before it and only then lets this one
  // be scheduled, and it leaves the lengths alone: they can be read while it
  // still runs.  One block waits for it in any case, so that this launch does
  // not end, and the next one on the stream not begin, before it.
  if (cta == 0 && row == 0) pdl_begin();
  if (threadIdx.x < 32) {
    const auto cta_begin = [](const PagedTotal& t, int64_t index) {
      return t.ranges.begin(kUnitWarps * index);
    };
    PagedStart start = {};
    const PagedTotal total = paged_start<kUnitTile, kUnitWarps, true>(
        a, grid_ctas, &start, [&](const PagedTotal& t) -> int64_t {
          return cta + 1 < t.ctas ? cta_begin(t, cta + 1) - 1 : -1;
        });
    int parts = 0, unit = 0;
    if (cta + 1 < total.ctas) {
      const int64_t at = cta_begin(total, cta + 1) - 1;  // the CTA's last tile
      const int tiles = key_tiles(start.length, kUnitTile);
      const TilePlace last = place_of(at, start.before, tiles, a.units.divisor);
      const int64_t unit_begin = at - last.tile;
      // Cut here, and not started by an earlier CTA.
      if (last.tile + 1 != tiles && unit_begin >= cta_begin(total, cta)) {
        unit = last.unit;
        parts = static_cast<int>(total.ranges.holder(unit_begin + tiles - 1) / kUnitWarps) - cta + 1;
      }
    }
    if (threadIdx.x == 0) found_sequence = start.sequence, found_unit = unit, found_parts = parts;
  }
  __syncthreads();
  const int parts = found_parts, sequence = found_sequence;
  if (parts == 0) return;
  const PagedUnit unit = paged_unit<kRows>(a, found_unit);
  if (row >= unit.rows) return;
  pdl_begin();  // the main launch's parts
  const auto part_row = [&](int p) {
    const int64_t slot = p == 0 ? 2 * static_cast<int64_t>(cta) + 1 : 2 * static_cast<int64_t>(cta + p);
    return slot * a.row_cap + row;
  };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += kJoinThreads)
    top = fmaxf(top, __ldcg(&a.partial_ml[part_row(p)]).x);
  top = warp_max(top);
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, warp_top[w]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, out[kHeld][kWidth] = {};
#pragma unroll 4
  for (int p = warp; p < parts; p += kJoinWarps) {
    const float2 ml = __ldcg(&a.partial_ml[part_row(p)]);
    const float f = paged_exp2(ml.x - base);
    sum = fmaf(f, ml.y, sum);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int d = (32 * i + lane) * kWidth;
      if (d >= a.head_dim) continue;
      float v[kWidth];
      ld_row_l2(a.partial + part_row(p) * a.head_dim + d, v);
#pragma unroll
      for (int e = 0; e < kWidth; ++e) out[i][e] = fmaf(f, v[e], out[i][e]);
    }
  }
  if (lane == 0) warp_sum[warp] = sum;
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
#pragma unroll
    for (int e = 0; e < kWidth; ++e) rows[warp][(32 * i + lane) * kWidth + e] = out[i][e];
  __syncthreads();
  for (int d = threadIdx.x; d < a.head_dim; d += kJoinThreads) {
    float l = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) l += warp_sum[w], o += rows[w][d];
    st_out(static_cast<T*>(a.out) +
               (static_cast<int64_t>(sequence) * a.heads + unit.first_head + row) * a.head_dim + d,
           top == -INFINITY ? 0.0f : __fdividef(o, l));
  }
}

template <typename T, int kUnitTile, int kUnitWarps, int kRows>
cudaError_t launch_join(const PagedArgs& a, int grid_ctas, cudaStream_t stream) {
  const dim3 grid(grid_ctas - 1, a.row_cap), block(kJoinThreads);
  if (a.head_dim % 4 == 0)
    return launch_pdl(paged_join_kernel<T, kUnitTile, kUnitWarps, kRows, 4>, grid, block, stream, a,
                      grid_ctas);
  return launch_pdl(paged_join_kernel<T, kUnitTile, kUnitWarps, kRows, 1>, grid, block, stream, a,
                    grid_ctas);
}

// Keys that a block table may have room for: a sequence's (positions are int,
// and tiles behind the last one are formed), and all sequences' together (the
// schedule counts tiles of 8 keys and more in 32 bits).
constexpr int64_t kPagedMaxLength = int64_t{1} << 30, kPagedMaxKeys = int64_t{1} << 34;

// The most CTAs of a launch; the workspace is sized for them.
inline int paged_grid_limit() { return 2 * sm_count(); }

// CTAs of a launch: at most `limit`, and no more than the longest batch that
// the block table can hold keeps busy.
inline int paged_grid(const PagedArgs& a, int limit, int tile, int warps, int unit_rows) {
  const int64_t capacity = static_cast<int64_t>(a.max_pages) * a.page_size.divisor;
  const int64_t tiles = capacity <= tile ? 1 : (capacity - 1) / tile + 1;
  const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads *
                        ((a.group + unit_rows - 1) / unit_rows);
  // The product may pass 63 bits; then only its comparison with the limit counts.
  const double total = static_cast<double>(tiles) * static_cast<double>(units);
  if (total >= static_cast<double>(limit) * warps) return limit;
  return active_ctas(tiles * units, limit, warps);
}

constexpr int kPagedMaxRows = 16;

// Floats of a CTA's parts put aside that do not fit beside 16 rows of more than
// 192 columns, four warps.
constexpr size_t kPagedHeadFloats = 4 * 16 * (kPagedMaxHeadDim + 4);
inline bool heads_in_scratch(int group, int head_dim) { return group > 8 && head_dim > 192; }

// Lays the scratch out; its size is that of the largest launch.
inline void paged_scratch(PagedArgs* a, int grid, int rows) {
  a->parts = make_fast_div((a->group + rows - 1) / rows);
  a->units = make_fast_div(a->kv_heads * a->parts.divisor);
  a->row_cap = a->group < rows ? a->group : rows;
  const int64_t slots = static_cast<int64_t>(grid) * 2 * a->row_cap;
  a->partial_ml = reinterpret_cast<float2*>(a->partial + slots * a->head_dim);
  a->aside = reinterpret_cast<float*>(a->partial_ml + slots);
}

inline size_t paged_scratch_bytes(int group, int head_dim) {
  const size_t rows = group < kPagedMaxRows ? group : kPagedMaxRows;
  return 2 * static_cast<size_t>(paged_grid_limit()) * rows *
             (sizeof(float) * head_dim + sizeof(float2)) +
         (heads_in_scratch(group, head_dim) ? sm_count() * kPagedHeadFloats * sizeof(float) : 0);
}

// The streaming kernels: head_dim a multiple of 16 bytes, addresses and strides
// too.
template <typename T>
int paged_attention_mma(const PagedArgs& a, cudaStream_t stream);
int paged_attention_f32(const PagedArgs& a, cudaStream_t stream);

}  // namespace opl
