// Attention of one new token per sequence over a paged key-value cache
// (opl_paged_attention_*), FP32 arithmetic, any head size up to 256, any
// grouping of query heads, any strides with a unit last one.
//
//   out[b, h] = sum_j p_j V_j,  p_j = exp(s_j - max s) / sum_i exp(s_i - max s),
//   s_j = scale * q[b, h] . K_j,  j < seq_lens[b], keys through the block table.
//
// This file has the entry points and the kernel for what the streaming kernels
// (paged_attention_mma.cu, paged_attention_f32.cu) do not take: rows that are no
// multiples of 16 bytes, or lie on other boundaries.
//
// The 32 lanes of a warp share a key: lane l holds elements l, l + 32, ... of
// the queries (up to 4 rows), of the key, of the value and of the output.  A
// warp takes 8 keys at a time; their scores are summed over the lanes by a
// transposing butterfly (about one shuffle a sum instead of five); one
// exponential a key and row; running maximum and sum (log2 domain) and the
// output in registers.  Loads are of one element: their issue bounds it.
#include "paged_attention.cuh"

namespace opl {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 8;  // keys of a warp's step

template <typename T>
__device__ __forceinline__ float ld_f32(const T* p);
template <>
__device__ __forceinline__ float ld_f32(const float* p) {
  return ld_stream(p);
}
template <>
__device__ __forceinline__ float ld_f32(const __half* p) {
  unsigned short b;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(b) : "l"(p));
  return __half2float(__ushort_as_half(b));
}
template <>
__device__ __forceinline__ float ld_f32(const __nv_bfloat16* p) {
  unsigned short b;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(b) : "l"(p));
  return __bfloat162float(__ushort_as_bfloat16(b));
}

constexpr int kElements = kPagedMaxHeadDim / 32;  // of a lane

// A row of a head into the lane's registers, zero past `dim` and where the row
// is not there.
template <typename T>
__device__ __forceinline__ void load_row(const T* row, int dim, int lane, float (&x)[kElements]) {
#pragma unroll
  for (int e = 0; e < kElements; ++e) {
    const int d = lane + 32 * e;
    x[e] = row != nullptr && d < dim ? ld_f32(row + d) : 0.0f;
  }
}

// Sums v[i] over the warp for each of kCount values (8, 16 or 32).  Afterwards
// v[0] of lane l is the sum of the value that the lane's bits spell from the
// top.
template <int kCount>
__device__ __forceinline__ void transpose_sum(float (&v)[kCount], int lane) {
  int count = kCount;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (count > 1) {
      count >>= 1;
#pragma unroll
      for (int i = 0; i < kCount / 2; ++i) {
        if (i >= count) continue;
        const bool upper = (lane & o) != 0;
        const float give = upper ? v[i] : v[i + count];
        const float keep = upper ? v[i + count] : v[i];
        v[i] = keep + __shfl_xor_sync(kFullMask, give, o);
      }
    } else {
      v[0] += __shfl_xor_sync(kFullMask, v[0], o);
    }
  }
}

constexpr int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads) paged_simt_kernel(const PagedArgs a) {
  constexpr int kSums = kTile * kRows;  // value index: row * kTile + key
  constexpr int E = kElements, kWidth = kPagedMaxHeadDim;
  static_assert(kSums <= 32, "a lane for each score");
  __shared__ float weights[kWarps][kRows][kTile];
  __shared__ float rescale[kWarps][kRows];
  __shared__ PagedParts<kWarps, kRows> parts;
  extern __shared__ __align__(16) float rows[];  // [2][kWarps][kRows][kWidth]
  float* const heads = rows + kWarps * kRows * kWidth;
  pdl_begin();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* q = static_cast<const T*>(a.q);
  const T* keys = static_cast<const T*>(a.k);
  const T* values = static_cast<const T*>(a.v);
  const int page_size = static_cast<int>(a.page_size.divisor);
  if (lane < 2) parts.records[warp][lane] = PartRecord{};
  const int64_t range = int64_t{kWarps} * blockIdx.x + warp;
  PagedStart start = {};
  const PagedTotal total = paged_start<kTile, kWarps, false>(
      a, gridDim.x, &start, [range](const PagedTotal& x) -> int64_t {
        const int64_t at = x.ranges.begin(range);
        return static_cast<int>(blockIdx.x) < x.ctas && at < x.tiles ? at : -1;
      });
  if (static_cast<int>(blockIdx.x) >= total.ctas) return;
  int64_t w = total.ranges.begin(range);
  const int64_t limit = total.ranges.begin(range + 1);
  const bool opens = w == total.ranges.begin(int64_t{kWarps} * blockIdx.x);
  int sequence = start.sequence;
  int64_t before = start.before;
  int reported = 0;

  // Which row's score this lane holds after transpose_sum: the value index is
  // spelled by the lane's bits from the top.
  constexpr int kLogSums = log2_of(kSums);
  const int index = lane >> (5 - kLogSums);
  const int my_row = index / kTile, my_key = index % kTile;

  while (w < limit) {
    const int raw_length = ld_int(a.seq_lens + sequence);
    const int length = readable_length(raw_length, a.max_pages, page_size);
    if (length != raw_length) reported = kBadLength;
    const int tiles = key_tiles(length, kTile);
    if (w >= (before + tiles) * a.units.divisor) {
      before += tiles;
      ++sequence;
      continue;
    }
    const TilePlace at = place_of(w, before, tiles, a.units.divisor);
    const int end = tiles - at.tile <= limit - w ? tiles : static_cast<int>(at.tile + (limit - w));
    w += end - at.tile;
    const PagedUnit unit = paged_unit<kRows>(a, at.unit);
    const int* table = a.block_table + sequence * a.table_row;
    const T* k_head = keys + unit.kv_head * a.k_head;
    const T* v_head = values + unit.kv_head * a.v_head;

    float qr[kRows][E], o[kRows][E];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      load_row<T>(
          r < unit.rows ? q + sequence * a.q_batch + (unit.first_head + r) * a.q_head : nullptr,
          a.head_dim, lane, qr[r]);
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;  // of my_row; l over my keys only
    bool has_keys = false;

    for (int tile = at.tile; tile < end; ++tile) {
      const int base = tile * kTile;
      // Lanes 0-7 place the tile's keys, lanes 8-15 its values.
      int64_t place = -1;
      {
        const int key = base + (lane & 7);
        if (lane < 16 && key < length) {
          const int index_in_row = static_cast<int>(fast_div(key, a.page_size));
          const int page = ld_int(table + index_in_row);
          const int inside = key - index_in_row * page_size;
          if (cache_page(page, a.pages))
            place = lane < 8 ? page * a.k_page + inside * a.k_token
                             : page * a.v_page + inside * a.v_token;
          else
            reported = kBadPage;
        }
      }
      has_keys |= __any_sync(kFullMask, place >= 0);
      float kr[kTile][E], vr[kTile][E];
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        const int64_t k_place = __shfl_sync(kFullMask, place, j);
        const int64_t v_place = __shfl_sync(kFullMask, place, 8 + j);
        load_row<T>(k_place >= 0 ? k_head + k_place : nullptr, a.head_dim, lane, kr[j]);
        load_row<T>(v_place >= 0 ? v_head + v_place : nullptr, a.head_dim, lane, vr[j]);
      }
      float s[kSums];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int j = 0; j < kTile; ++j) {
          float dot = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) dot = fmaf(qr[r][e], kr[j][e], dot);
          s[r * kTile + j] = dot;
        }
      transpose_sum(s, lane);
      const bool there = __shfl_sync(kFullMask, place, my_key) >= 0;
      const float score = there ? s[0] * a.scale_log2 : -INFINITY;
      float top = score;
      // The lanes that hold one row differ in these bits.
      constexpr int kRowLanes = 8;
      constexpr int kFirst = 4 / kRows;
#pragma unroll
      for (int x = 1; x < kRowLanes; x <<= 1)
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, x * kFirst));
      const float m_new = fmaxf(m, top);
      const float base_m = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: all weights 0
      const float alpha = paged_exp2(m - base_m);
      __syncwarp();  // the previous tile's weights have been read
      const float weight = paged_exp2(score - base_m);
      weights[warp][my_row][my_key] = weight;
      if (my_key == 0) rescale[warp][my_row] = alpha;
      l = l * alpha + weight;
      m = m_new;
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float alpha_r = rescale[warp][r];
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] *= alpha_r;
#pragma unroll
        for (int j = 0; j < kTile; ++j) {
          const float p = weights[warp][r][j];
#pragma unroll
          for (int e = 0; e < E; ++e) o[r][e] = fmaf(p, vr[j][e], o[r][e]);
        }
      }
    }

    // Every lane that holds a row has its maximum; the sum is over the lanes
    // that hold different keys of it.
    constexpr int kRowLanes = 8;
    constexpr int kFirst = 4 / kRows;
#pragma unroll
    for (int x = 1; x < kRowLanes; x <<= 1) l += __shfl_xor_sync(kFullMask, l, x * kFirst);
    constexpr int kLanesOfRow = 32 / kRows;  // lane of row r: the first of these
    if (at.tile == 0 && end == tiles) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float sum = __shfl_sync(kFullMask, l, r * kLanesOfRow);
        if (r >= unit.rows) continue;
        T* const dst = static_cast<T*>(a.out) +
                       (static_cast<int64_t>(sequence) * a.heads + unit.first_head + r) * a.head_dim;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int d = lane + 32 * e;
          if (d < a.head_dim) st_out(dst + d, has_keys ? o[r][e] / sum : 0.0f);
        }
      }
      continue;
    }
    const int kind = at.tile == 0 ? kTail : kHead;
    const bool aside = w < limit;
    float* const part = (aside ? heads : rows) + warp * kRows * kWidth;
    if (lane % kLanesOfRow == 0 && my_row < unit.rows) {
      parts.m[warp][kind][my_row] = fmaxf(m, least_maximum(has_keys));
      parts.l[warp][kind][my_row] = l;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= unit.rows) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + 32 * e;
        if (d < a.head_dim) part[r * kWidth + d] = o[r][e];
      }
    }
    if (lane == 0)
      parts.records[warp][kind] = PartRecord{sequence, at.unit, tiles,  at.tile,
                                             end,      opens && kind == kHead, aside};
  }
  if (reported != 0) watchdog_trip(a.watchdog, reported);
  __syncthreads();
  paged_merge<T, kWarps, kRows, kRows * kWidth, kWidth, 1>(a, parts, rows, heads);
}

template <typename T, int kRows>
int launch_simt(PagedArgs a, cudaStream_t stream) {
  const int grid = paged_grid(a, paged_grid_limit(), kTile, kWarps, kRows);
  paged_scratch(&a, grid, kRows);
  constexpr size_t kShared = sizeof(float) * 2 * kWarps * kRows * kPagedMaxHeadDim;
  const cudaError_t allowed =
      cudaFuncSetAttribute(paged_simt_kernel<T, kRows>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(kShared));
  if (allowed != cudaSuccess) return allowed;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kShared;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  cudaError_t error = cudaLaunchKernelEx(&config, paged_simt_kernel<T, kRows>, a);
  if (error == cudaSuccess && grid > 1)
    error = launch_join<T, kTile, kWarps, kRows>(a, grid, stream);
  return error != cudaSuccess ? error : cudaGetLastError();
}

bool aligned_rows(const PagedArgs& a, size_t element) {
  const int vector = 16 / static_cast<int>(element);
  const int64_t strides[] = {a.q_batch, a.q_head, a.k_page, a.k_token, a.k_head,
                             a.v_page,  a.v_token, a.v_head, a.head_dim};
  for (int64_t s : strides)
    if (s % vector != 0) return false;
  for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.out)})
    if (!aligned16(p)) return false;
  return true;
}

template <typename T>
int paged_attention(const void* q, int64_t q_batch, int64_t q_head, const opl_kv_cache* cache,
                    const int* block_table, int64_t table_row, int max_pages, const int* seq_lens,
                    void* out, int batch, int heads, float scale, void* workspace,
                    size_t workspace_bytes, cudaStream_t stream) {
  if (q == nullptr || cache == nullptr || cache->k == nullptr || cache->v == nullptr ||
      block_table == nullptr || seq_lens == nullptr || out == nullptr || workspace == nullptr ||
      batch <= 0 || heads <= 0 || max_pages <= 0 || cache->pages <= 0 || cache->page_size <= 0 ||
      cache->kv_heads <= 0 || heads % cache->kv_heads != 0 || cache->head_dim <= 0 ||
      cache->head_dim > kPagedMaxHeadDim || !(scale - scale == 0.0f) ||
      reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0 ||
      static_cast<int64_t>(max_pages) * cache->page_size > kPagedMaxLength ||
      static_cast<int64_t>(max_pages) * cache->page_size > kPagedMaxKeys / batch)
    return cudaErrorInvalidValue;
  size_t needed = 0;
  const int status = opl_paged_attention_workspace(heads, cache->kv_heads, cache->head_dim, &needed);
  if (status != cudaSuccess) return status;
  if (workspace_bytes < needed) return cudaErrorInvalidValue;
  PagedArgs a = {};
  a.q = q;
  a.k = cache->k;
  a.v = cache->v;
  a.out = out;
  a.q_batch = q_batch;
  a.q_head = q_head;
  a.k_page = cache->k_page;
  a.k_token = cache->k_token;
  a.k_head = cache->k_head;
  a.v_page = cache->v_page;
  a.v_token = cache->v_token;
  a.v_head = cache->v_head;
  a.block_table = block_table;
  a.table_row = table_row;
  a.seq_lens = seq_lens;
  a.pages = cache->pages;
  a.page_size = make_fast_div(cache->page_size);
  a.max_pages = max_pages;
  a.batch = batch;
  a.heads = heads;
  a.kv_heads = cache->kv_heads;
  a.head_dim = cache->head_dim;
  a.group = heads / cache->kv_heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.partial = static_cast<float*>(workspace);
  a.watchdog = watchdog_word();
  if (a.watchdog == nullptr) return cudaErrorInvalidDevice;
  if (aligned_rows(a, sizeof(T))) {
    if constexpr (sizeof(T) == 4)
      return paged_attention_f32(a, stream);
    else
      return paged_attention_mma<T>(a, stream);
  }
  return a.group == 1 ? launch_simt<T, 1>(a, stream) : launch_simt<T, 4>(a, stream);
}

}  // namespace

}  // namespace opl

extern "C" {

int opl_paged_attention_workspace(int heads, int kv_heads, int head_dim, size_t* bytes) {
  if (bytes == nullptr || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0 ||
      head_dim > opl::kPagedMaxHeadDim)
    return cudaErrorInvalidValue;
  *bytes = opl::paged_scratch_bytes(heads / kv_heads, head_dim);
  return cudaSuccess;
}

#define OPL_PAGED_ENTRY(SUFFIX, ABI_T, T)                                                          \
  int opl_paged_attention_##SUFFIX(const ABI_T* q, int64_t q_batch, int64_t q_head,                \
                                   const opl_kv_cache* cache, const int* block_table,              \
                                   int64_t table_row, int max_pages, const int* seq_lens,          \
                                   ABI_T* out, int batch, int heads, float scale, void* workspace, \
                                   size_t workspace_bytes, opl_stream_t stream) {                  \
    return opl::paged_attention<T>(q, q_batch, q_head, cache, block_table, table_row, max_pages,   \
                                   seq_lens, out, batch, heads, scale, workspace, workspace_bytes, \
                                   stream);                                                        \
  }

OPL_PAGED_ENTRY(f32, float, float)
OPL_PAGED_ENTRY(f16, opl_half_t, __half)
OPL_PAGED_ENTRY(bf16, opl_bf16_t, __nv_bfloat16)

}  // extern "C"
