// Streaming frame of the paged decode attention kernels: every warp reads its
// range of key tiles through a ring of stages in shared memory, and a Policy
// does the arithmetic of a tile (paged_attention_mma.cu: 16-bit types on the
// tensor cores; paged_attention_f32.cu: FP32).
//
// A warp has a ring of its own, a tile of keys and a tile of values a stage,
// and never waits for another warp:
//
// * The tiles come by TMA (a box of kTile tokens x 128 bytes of one head, all
//   pieces of 128 bytes in one copy, 128-byte swizzle; boxes of 8 tokens when
//   kTile is no divisor of the page size).  Copies by the lanes (cp.async),
//   which every page size and stride allows, put the same layout there but take
//   an instruction per 512 bytes: with 131071 keys, 32/8 heads of 128 in BF16,
//   their issue alone bounds the kernel (106 us with no arithmetic, 138 us when
//   a group of eight lanes does not cover 128 bytes of a row; TMA 87 us with it).
// * Two stages of 8 KB for each of 8 warps are enough: a batch of 128 sequences
//   up to 8191 keys takes 306 to 323 us on different boards, the copy rate; with
//   three stages, when it took 318, 341.
// * Two cursors walk over the tiles, one for copies and one for arithmetic, so
//   that the copies run on across the ends of sequences and heads.
//
// What bounds long sequences after that is that the SMs do not stream at one
// rate: 40 of the 148 (four groups of ten) take 149,000 cycles for a range that
// the others read in 125,000, and ranges are cut equal.  Short ones are bound by
// the chain from lengths over block table and keys to the output, whose code
// runs once: it is kept short, and rolled.
#pragma once

#include <atomic>

#include "paged_attention.cuh"
#include "tc_common.cuh"
#include "tmap.cuh"

namespace opl {

// 16 bytes to shared memory, zeros when `there` is false (nothing is read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ uint4 ld_shared(uint32_t src) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(src)
               : "memory");
  return r;
}

// How the tensor maps of the caches are laid out: dimensions (columns of a
// 128-byte piece, token, piece, head, page).
struct MapOrder {
  int boxes;   // of a tile: one of kTile tokens, or several of 8
  int copies;  // of a box: all pieces at once, or each by itself where a box is
               // not the whole tile or the last piece is short (the map then has
               // one piece, of head_dim columns)
};

// Sizes of a Policy's ring.  kDim: head_dim rounded up.
template <typename Policy, int kWarps, int kStages>
struct Ring {
  using T = typename Policy::T;
  static constexpr int kKeyBytes = Policy::kTile * Policy::kDim * static_cast<int>(sizeof(T));
  static constexpr int kStageBytes = 2 * kKeyBytes;
  static constexpr int kBytes = kStages * kStageBytes;  // of a warp
  static constexpr int kPitch = Policy::kDim + 4;       // of a merged row, in floats
  // A part put aside, in shared memory but for 16 rows of 256 columns, whose
  // kernel spills and is slower with less L1 (16/1 heads of 256: 31.0 us, against
  // 34.3 with the parts in shared memory).
  static constexpr bool kSharedHeads = Policy::kRows * Policy::kDim <= 16 * 192;
  static constexpr int kHeadBytes = kSharedHeads ? Policy::kRows * kPitch * 4 : 0;
  static constexpr size_t kShared =
      1024 + static_cast<size_t>(kWarps) * (kBytes + Policy::kWarpShared + kHeadBytes);
  static_assert(kStageBytes % 1024 == 0 && Policy::kWarpShared % 16 == 0, "alignment");
  static_assert(Policy::kRows * kPitch * 4 <= kBytes, "a warp merges through its own ring");
  static_assert(kShared <= 220 * 1024, "beside the static arrays");
  static_assert(Policy::kRows <= kPagedMaxRows, "paged_scratch_bytes");
  static_assert(kSharedHeads || kWarps * Policy::kRows * kPitch <= static_cast<int>(kPagedHeadFloats),
                "kPagedHeadFloats");
};

// Copies are made by the TMA unit, or by the lanes (kTma false).
template <typename Policy, bool kTma, int kWarps, int kStages>
__global__ void __launch_bounds__(32 * kWarps, 1)
    paged_stream_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map, const MapOrder order) {
  using S = Ring<Policy, kWarps, kStages>;
  using T = typename Policy::T;
  constexpr int kTile = Policy::kTile, kRows = Policy::kRows;
  constexpr int kWidth = 128 / static_cast<int>(sizeof(T));  // columns of a piece
  constexpr int kPieceBytes = kTile * 128;
  constexpr int kPieces = Policy::kDim / kWidth;
  constexpr uint32_t kAll = (1u << kTile) - 1;
  extern __shared__ unsigned char shared[];
  __shared__ PagedParts<kWarps, kRows> parts;
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int abort_wait;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned char* const rings = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<std::uintptr_t>(shared) + 1023) & ~static_cast<std::uintptr_t>(1023));
  unsigned char* const ring = rings + warp * S::kBytes;
  const auto heads = [&] {
    return S::kSharedHeads
               ? reinterpret_cast<float*>(rings + kWarps * (S::kBytes + Policy::kWarpShared))
               : a.aside + blockIdx.x * kPagedHeadFloats;
  };
  if constexpr (kTma) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) tc::mbar_init(&full[warp][i], 1);
      tc::fence_barrier_init();
      if (warp == 0) {
        abort_wait = 0;
        tc::prefetch_tmap(&k_map);
        tc::prefetch_tmap(&v_map);
      }
    }
  }
  __syncthreads();
  pdl_begin();

  const int page_size = static_cast<int>(a.page_size.divisor);
  if (lane < 2) parts.records[warp][lane] = PartRecord{};
  const int64_t range = int64_t{kWarps} * blockIdx.x + warp;
  PagedStart start;
  const PagedTotal total = paged_start<kTile, kWarps, false>(
      a, gridDim.x, &start, [range](const PagedTotal& x) -> int64_t {
        const int64_t at = x.ranges.begin(range);
        return static_cast<int>(blockIdx.x) < x.ctas && at < x.tiles ? at : -1;
      });
  if (static_cast<int>(blockIdx.x) >= total.ctas) return;
  const int64_t w = total.ranges.begin(range);
  const bool opens = w == total.ranges.begin(int64_t{kWarps} * blockIdx.x);
  int64_t to_fetch = total.ranges.begin(range + 1) - w, to_read = to_fetch;
  int reported = 0;
  int slot_in = 0, slot_out = 0;  // ring stages being filled and read
  uint32_t parity = 0;            // of the stage being read

  const uint32_t ring_address = tc::smem_u32(ring);

  // Two cursors walk over the warp's tiles: `in`, the next one to be fetched,
  // and `out`, the one being read.  The length of the next sequence is loaded
  // while this one lasts.
  struct Cursor {
    int sequence, unit, tile, tiles, length, next_length;
  };
  const int units = static_cast<int>(a.units.divisor);
  const auto load_length = [&](int sequence) {
    return sequence < a.batch ? ld_int(a.seq_lens + sequence) : 0;
  };
  const auto enter = [&](Cursor& c, int raw) {
    c.length = readable_length(raw, a.max_pages, page_size);
    if (c.length != raw) reported = kBadLength;
    c.tiles = key_tiles(c.length, kTile);
    c.next_length = load_length(c.sequence + 1);
  };
  const auto advance = [&](Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.unit < units) return;
    c.unit = 0;
    ++c.sequence;
    enter(c, c.next_length);
  };
  Cursor in = {};
  if (to_read > 0) {
    if (start.raw_length != start.length) reported = kBadLength;
    in.sequence = start.sequence;
    in.length = start.length;
    in.tiles = key_tiles(in.length, kTile);
    in.next_length = load_length(in.sequence + 1);
    const TilePlace p = place_of(w, start.before, in.tiles, units);
    in.unit = p.unit;
    in.tile = p.tile;
  }
  Cursor out = in;

  // Block-table entries are loaded for a batch of tiles of one unit, a batch
  // ahead: with the TMA unit a lane for each 8 keys, else one for each key.
  constexpr int kKeysPerLane = kTma ? 8 : 1, kBatchLanes = kTile / kKeysPerLane;
  constexpr int kBatch = 32 / kBatchLanes;
  struct Batch {
    int tile, left, length, kv_head;
    int page, inside;  // of this lane's key; page -1: no key
    uint32_t whole;    // bit of each lane: its keys' page is in the cache
  };
  const auto fetch = [&]() {
    Batch f = {};
    if (to_fetch > 0) {
      f.tile = in.tile;
      f.left = min(min(kBatch, in.tiles - in.tile), static_cast<int>(min(to_fetch, int64_t{kBatch})));
      f.length = in.length;
      f.kv_head = static_cast<int>(fast_div(in.unit, a.parts));
      const int key = (in.tile + lane / kBatchLanes) * kTile + lane % kBatchLanes * kKeysPerLane;
      const int row = static_cast<int>(fast_div(key, a.page_size));
      f.inside = key - row * page_size;
      f.page = -1;
      if (key < in.length) f.page = ld_int(a.block_table + in.sequence * a.table_row + row);
      to_fetch -= f.left;
      in.tile += f.left - 1;
      advance(in);
    }
    return f;
  };
  Batch batch = {}, next_batch = {};
  int batch_lane = 0;
  // Copies a tile into the next stage; bit j of the result: key j is there.
  const auto issue = [&]() -> uint32_t {
    uint32_t there = 0;
    while (batch.left == 0 && (next_batch.left > 0 || to_fetch > 0)) {
      batch = next_batch;
      next_batch = fetch();
      batch_lane = lane % kBatchLanes;
      const bool known = (batch.tile + lane / kBatchLanes) * kTile +
                             lane % kBatchLanes * kKeysPerLane < batch.length;
      const bool ok = cache_page(batch.page, a.pages);
      if (known && !ok) reported = kBadPage;
      if (!known || !ok) batch.page = -1;
      batch.whole = __ballot_sync(kFullMask, batch.page >= 0);
    }
    if (batch.left > 0) {
      const int page = __shfl_sync(kFullMask, batch.page, batch_lane);
      const int inside = __shfl_sync(kFullMask, batch.inside, batch_lane);
      // The bits of this tile's lanes.
      const uint32_t pages = batch.whole >> (batch_lane - lane % kBatchLanes);
      batch_lane += kBatchLanes;
      --batch.left;
      const int left = batch.length - batch.tile++ * kTile;
      if constexpr (kTma) {
        there = left >= kTile ? kAll : (1u << left) - 1;
#pragma unroll
        for (int half = 0; half < kBatchLanes; ++half)
          if ((pages >> half & 1u) == 0) there &= ~(0xffu << (8 * half));
        uint64_t* const bar = &full[warp][slot_in];
        if (lane == 0) tc::mbar_expect_tx(bar, S::kStageBytes);
        __syncwarp();
        if (lane < order.boxes) {
          // A box that holds no key lies past the last page: zeros.
          const int p = page >= 0 ? page : static_cast<int>(a.pages);
          unsigned char* dst = ring + slot_in * S::kStageBytes + lane * 1024;
#pragma unroll 1
          for (int c = 0; c < order.copies; ++c, dst += kPieceBytes) {
            tc::tma_load_5d(dst, &k_map, kWidth * c, inside, 0, batch.kv_head, p, bar);
            tc::tma_load_5d(dst + S::kKeyBytes, &v_map, kWidth * c, inside, 0, batch.kv_head, p, bar);
          }
        }
      } else {
        const int64_t place =
            page < 0    ? -1
            : lane < 16 ? page * a.k_page + inside * a.k_token + batch.kv_head * a.k_head
                        : page * a.v_page + inside * a.v_token + batch.kv_head * a.v_head;
        there = pages & kAll;
        // Eight lanes copy 128 bytes of one row.
        const int piece = lane & 7;
        const uint32_t dst = ring_address + slot_in * S::kStageBytes;
        constexpr int kLoads = kTile / 4, kElements = kWidth / 8;  // of 16 bytes
#pragma unroll
        for (int s = 0; s < 2 * kLoads; ++s) {
          const bool is_key = s < kLoads;
          const int row = 4 * (s % kLoads) + (lane >> 3);
          const int64_t at = __shfl_sync(kFullMask, place, (is_key ? 0 : 16) + row);
          const T* const src =
              static_cast<const T*>(is_key ? a.k : a.v) + (at >= 0 ? at : 0) + kElements * piece;
          const uint32_t to = dst + (is_key ? 0 : S::kKeyBytes) + row * 128 + (piece ^ (row & 7)) * 16;
#pragma unroll
          for (int c = 0; c < kPieces; ++c)
            copy16(to + c * kPieceBytes, src + kWidth * c,
                   at >= 0 && kWidth * c + kElements * piece < a.head_dim);
        }
      }
      if (++slot_in == kStages) slot_in = 0;
    }
    if constexpr (!kTma) copy_commit();
    return there;
  };

  Policy policy;
  policy.init(lane, reinterpret_cast<float*>(rings + kWarps * S::kBytes +
                                             warp * Policy::kWarpShared));
  int begin = out.tile;  // of the segment
  // The queries of the next segment are loaded during this one.
  const auto fetch_next_query = [&]() {
    const bool same = out.unit + 1 < units;
    if (same || out.sequence + 1 < a.batch)
      policy.fetch_query(a, same ? out.sequence : out.sequence + 1, same ? out.unit + 1 : 0);
  };
  if (to_read > 0) policy.fetch_query(a, out.sequence, out.unit);
  bool fresh = true;  // the next tile read is its segment's first

  // Step s copies tile s and, once kStages - 1 tiles are on their way, reads
  // tile s - (kStages - 1).  (One loop for the first steps and the others:
  // code that runs once costs its instruction fetches, about as long as the
  // copies take.)
  uint32_t there[kStages] = {};
  int early = kStages - 1;
  while (to_read > 0) {
    __syncwarp();  // every lane has read the stage that is filled next
#pragma unroll
    for (int x = 0; x + 1 < kStages; ++x) there[x] = there[x + 1];
    there[kStages - 1] = issue();
    if (early > 0) {
      --early;
      continue;
    }
    if constexpr (kTma) {
      if (!tc::mbar_wait_warp(&full[warp][slot_out], parity, &abort_wait, a.watchdog,
                              tc::kWatchdogPaged)) {
        // Give the other copies in flight the same time to land and stop; the
        // output is not valid and the watchdog says so.
        for (int x = 1; x < kStages && x < to_read; ++x) {
          const int slot = (slot_out + x) % kStages;
          volatile int alone = 0;
          tc::mbar_wait(&full[warp][slot], slot < slot_out ? parity ^ 1u : parity, &alone,
                        a.watchdog, tc::kWatchdogPaged);
        }
        break;
      }
    } else {
      copy_wait<kStages - 1>();
      __syncwarp();  // what the other lanes copied
    }
    const uint32_t stage = ring_address + slot_out * S::kStageBytes;
    if (++slot_out == kStages) slot_out = 0, parity ^= 1u;

    if (fresh) {
      fresh = false;
      policy.start(a, out.sequence, out.unit);
      fetch_next_query();
    }
    policy.step(a, stage, stage + S::kKeyBytes, there[0]);

    --to_read;
    if (out.tile + 1 < out.tiles && to_read > 0) {
      ++out.tile;
      continue;
    }

    // The segment ends.  A part goes to the ring, which is empty, when the warp
    // is done, else aside.
    const PagedUnit unit = paged_unit<kRows>(a, out.unit);
    const bool whole = begin == 0 && out.tile + 1 == out.tiles;
    const bool aside = to_read > 0;
    const int kind = begin == 0 ? kTail : kHead;
    if constexpr (!kTma) {
      if (!whole) copy_wait<0>();
    }
    __syncwarp();  // every lane has read its last stage
    const bool odd = policy.settle();
    const auto part = [&] {
      return aside ? heads() + warp * kRows * S::kPitch : reinterpret_cast<float*>(ring);
    };
    if (whole)
      policy.finish_whole(a, unit, out.sequence, out.length == 0);
    else
      policy.finish_part(a, unit, part(), S::kPitch, parts.m[warp][kind], parts.l[warp][kind]);
    if (odd && out.length != 0) {
      const int first = begin * kTile, end = min(out.length, (out.tile + 1) * kTile);
      T* const rows = static_cast<T*>(a.out) +
                      (static_cast<int64_t>(out.sequence) * a.heads + unit.first_head) * a.head_dim;
      if constexpr (Policy::kInfiniteValues)
        policy.infinite_values(a, unit, out.sequence, first, end, [&](int row, int column, float x) {
          if (whole)
            st_out(rows + row * a.head_dim + column, x);
          else
            part()[row * S::kPitch + column] = x;
        });
      const bool keys = any_page(a, out.sequence, first, end);
      __syncwarp();  // what the other lanes have written
      if (whole && !keys) {
        for (int i = lane; i < unit.rows * a.head_dim; i += 32) st_out(rows + i, 0.0f);
      } else if (!whole && lane < unit.rows) {
        parts.m[warp][kind][lane] = fmaxf(parts.m[warp][kind][lane], least_maximum(keys));
      }
    }
    if (!whole && lane == 0)
      parts.records[warp][kind] = PartRecord{out.sequence, out.unit,     out.tiles, begin,
                                             out.tile + 1, opens && kind == kHead, aside};
    if (to_read > 0) {
      advance(out);
      begin = 0;
      fresh = true;
    }
  }
  if (reported != 0) watchdog_trip(a.watchdog, reported);
  __syncthreads();
  paged_merge<T, kWarps, kRows, S::kBytes / 4, S::kPitch, 4>(
      a, parts, reinterpret_cast<const float*>(rings), heads());
}

// Encodes a cache for the TMA unit; false when its layout does not allow it.
// `pieces`: of a stage's row; those past head_dim are filled with zeros.
template <typename T>
bool cache_map(CUtensorMap* map, const PagedArgs& a, const void* base, int64_t page, int64_t token,
               int64_t head, const MapOrder& order, int tile, int pieces) {
  constexpr int kWidth = 128 / static_cast<int>(sizeof(T)), kAligned = 16 / static_cast<int>(sizeof(T));
  const bool together = order.copies == 1;
  const uint64_t extent[5] = {
      static_cast<uint64_t>(together && a.head_dim > kWidth ? kWidth : a.head_dim),
      a.page_size.divisor,
      static_cast<uint64_t>(together ? (a.head_dim + kWidth - 1) / kWidth : 1),
      static_cast<uint64_t>(a.kv_heads), static_cast<uint64_t>(a.pages)};
  int64_t stride[4] = {token, kWidth, head, page};
  const uint32_t box[5] = {static_cast<uint32_t>(kWidth), static_cast<uint32_t>(tile / order.boxes),
                           static_cast<uint32_t>(together ? pieces : 1), 1, 1};
  uint64_t bytes[4];
  for (int i = 0; i < 4; ++i) {
    // A dimension of one element may come with any stride.
    if (extent[i + 1] == 1) stride[i] = kAligned;
    if (stride[i] <= 0 || stride[i] >= (int64_t{1} << 37)) return false;
    bytes[i] = static_cast<uint64_t>(stride[i]) * sizeof(T);
  }
  const CUtensorMapDataType type = sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return encode_tmap(map, type, 5, base, extent, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B) ==
         cudaSuccess;
}

template <typename Policy, bool kTma, int kWarps, int kStages>
int launch_stream(const PagedArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map,
                  const MapOrder& order, int grid, cudaStream_t stream) {
  constexpr auto kernel = paged_stream_kernel<Policy, kTma, kWarps, kStages>;
  constexpr size_t kShared = Ring<Policy, kWarps, kStages>::kShared;
  // Once a device: the call takes a microsecond of the host's time.
  static std::atomic<uint64_t> allowed{0};
  const int device = current_device();
  const uint64_t bit = device >= 0 && device < 64 ? uint64_t{1} << device : 0;
  cudaError_t error = cudaSuccess;
  if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
    error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(kShared));
    if (error != cudaSuccess) return error;
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(32 * kWarps);
  config.dynamicSmemBytes = kShared;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  error = cudaLaunchKernelEx(&config, kernel, a, k_map, v_map, order);
  if (error == cudaSuccess && grid > 1)
    error = launch_join<typename Policy::T, Policy::kTile, kWarps, Policy::kRows>(a, grid, stream);
  return error != cudaSuccess ? error : cudaGetLastError();
}

// One CTA a SM, copies by the TMA unit where the caches' layout allows it.
template <typename Policy, int kWarps, int kStages>
int paged_stream(PagedArgs a, cudaStream_t stream) {
  using T = typename Policy::T;
  constexpr int kTile = Policy::kTile, kWidth = 128 / static_cast<int>(sizeof(T));
  if (a.pages > 0x7fffffff) a.pages = 0x7fffffff;  // as far as block-table entries reach
  const int grid = paged_grid(a, sm_count(), kTile, kWarps, Policy::kRows);
  paged_scratch(&a, grid, Policy::kRows);
  CUtensorMap k_map = {}, v_map = {};
  constexpr int kPieces = Policy::kDim / kWidth;
  MapOrder order = {a.page_size.divisor % kTile == 0 ? 1 : kTile / 8, kPieces};
  if (order.boxes == 1 && a.head_dim % kWidth == 0) order.copies = 1;
  if (a.page_size.divisor % 8 == 0 &&
      cache_map<T>(&k_map, a, a.k, a.k_page, a.k_token, a.k_head, order, kTile, kPieces) &&
      cache_map<T>(&v_map, a, a.v, a.v_page, a.v_token, a.v_head, order, kTile, kPieces))
    return launch_stream<Policy, true, kWarps, kStages>(a, k_map, v_map, order, grid, stream);
  return launch_stream<Policy, false, kWarps, kStages>(a, k_map, v_map, order, grid, stream);
}

}  // namespace opl
