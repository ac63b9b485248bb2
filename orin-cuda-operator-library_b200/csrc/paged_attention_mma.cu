// Paged decode attention on 16-bit caches (see paged_attention.cu for the
// operator): a stream over the keys and values at HBM speed, with the products
// on warp-level tensor-core instructions.
//
// Bound by HBM: 4 operations per cached element and query head, so a group of
// 8 query heads asks for 8 operations a byte, 52 TFLOP/s at 6.5 TB/s -- more
// than FP32 units can give beside the rest, little for mma.sync (m16n8k16).
// tcgen05 has nothing to add: its smallest tile has 64 rows, its operands have
// to be written to shared memory in a swizzled layout (with V transposed), and
// the rate is not what bounds.
//
// One warp owns 16 keys at a time and a ring of stages, a tile of keys and a
// tile of values each; it never waits for another warp:
//
// * The tiles come by TMA (a box of 16 tokens x 64 columns of one head, 128-byte
//   swizzle; two boxes of 8 tokens when 16 is no divisor of the page size).
//   Copies by the lanes (cp.async), which every page size and stride allows,
//   put the same layout there but take an instruction per 512 bytes and lane
//   group: with 131071 keys, 32/8 heads of 128 in BF16, their issue alone
//   bounds the kernel (106 us with no arithmetic, 138 us when a group of eight
//   lanes does not cover 128 bytes of a row; TMA 97 us with it).  8 warps x 3
//   stages keep 192 KB in flight per SM (5 x 5 or 6 x 4: 99-105 us).
// * A contraction may run over its index in any order, so operands are read
//   from that layout by conflict-free 128-bit loads, without ldmatrix.
//   S = Q K^T: lane (g, t) of an m16n8k16 B operand holds row g (key g); two
//   instructions take 8 consecutive elements of it, those at 16t + 8 (j & 1)
//   of the 64-column box; Q is loaded in the same order.  O = P V: the operand
//   pairs two keys of one column, so the lane loads 8 consecutive columns of
//   keys 2t, 2t+1, 2t+8, 2t+9 -- the keys whose weights the S accumulator left
//   in this lane -- and one byte permute a register pairs them; instruction e
//   of 8 then computes columns 8n + e of the box, which lands 8 consecutive
//   columns of a row in one lane.
// * The weights enter P V as the sum of two 16-bit values, so that their
//   rounding (2^-9 in BF16, as much as the result's own) does not show.  With
//   up to 8 query heads a unit the second value rides in the 8 rows of the
//   operand that are otherwise empty.
//
// Running maximum, sum and output are FP32 in registers; the warps of a CTA
// merge at the end of a segment, and cut units are joined by a second launch.
#include "paged_attention.cuh"
#include "tc_common.cuh"
#include "tmap.cuh"

namespace opl {

namespace {

constexpr int kTile = 16;

template <typename T>
struct Mma;
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  // (x, y) rounded, x in the low half; and what the rounding left.
  static __device__ __forceinline__ uint32_t split(float x, float y, uint32_t* rest) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 back = __half22float2(h);
    const __half2 r = __floats2half2_rn(x - back.x, y - back.y);
    *rest = *reinterpret_cast<const uint32_t*>(&r);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t split(float x, float y, uint32_t* rest) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 back = __bfloat1622float2(h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - back.x, y - back.y);
    *rest = *reinterpret_cast<const uint32_t*>(&r);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

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

// The low (or high) halves of two words, a's first.
template <bool kHigh>
__device__ __forceinline__ uint32_t pair_halves(uint32_t a, uint32_t b) {
  return __byte_perm(a, b, kHigh ? 0x7632 : 0x5410);
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// kDim: head_dim rounded up to a multiple of 64.  kRows: 8 or 16 query heads
// a unit.
template <typename T, int kDim, int kRows, int kWarps, int kStages>
struct Shape {
  static constexpr int kKeyBytes = kTile * kDim * 2;
  static constexpr int kStageBytes = 2 * kKeyBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;  // of a warp
  static constexpr int kPitch = kDim + 4;  // of a merged row, in floats
  static constexpr size_t kShared = 1024 + static_cast<size_t>(kWarps) * kRingBytes;
  static_assert(kRows * kPitch * 4 <= kRingBytes, "a warp merges through its own ring");
  static_assert(kShared <= 222 * 1024, "beside the static arrays");
};

// How the tensor maps of the caches are laid out: dimensions (64 columns,
// token, 64-column piece, head, page).
struct MapOrder {
  int boxes;   // of a tile: one of 16 tokens, or two of 8
  int copies;  // of a box: all pieces at once, or each by itself where a box is
               // not 16 tokens or the last piece is short (the map then has one
               // piece, of head_dim columns)
};

// Copies are made by the TMA unit, or by the lanes (kTma false).
template <typename T, int kDim, int kRows, bool kTma, int kWarps, int kStages>
__global__ void __launch_bounds__(32 * kWarps, 1)
    paged_mma_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map, const MapOrder order) {
  using S = Shape<T, kDim, kRows, kWarps, kStages>;
  constexpr int kHalves = kRows / 8;  // row groups of the S accumulator in use
  extern __shared__ unsigned char shared[];
  __shared__ PagedParts<kWarps, kRows> parts;
  __shared__ uint64_t full[kWarps][kStages];
  __shared__ int abort_wait;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* const rings = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<std::uintptr_t>(shared) + 1023) & ~static_cast<std::uintptr_t>(1023));
  unsigned char* const ring = rings + warp * S::kRingBytes;
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

  const T* q = static_cast<const T*>(a.q);
  const int page_size = static_cast<int>(a.page_size.divisor);
  if (lane < 2) parts.records[warp][lane] = PartRecord{};
  const int64_t range = int64_t{kWarps} * blockIdx.x + warp;
  PagedStart start;
  const PagedTotal total = paged_start<kTile, kWarps>(
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

  // Where this lane's pieces lie in a stage (see the layout above).
  const uint32_t k_piece = g * 128 + (2 * t ^ g) * 16;
  const uint32_t v_piece = S::kKeyBytes + 2 * t * 128 + (g ^ 2 * t) * 16;
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
  // ahead: with the TMA unit 16 tiles of two boxes of 8 keys (one of 16: the
  // even lanes), a lane each; else two tiles, a lane for each key.
  constexpr int kBatch = kTma ? 16 : 2;
  constexpr int kBatchLanes = 32 / kBatch, kKeysPerLane = kTile / kBatchLanes;
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
        there = left >= kTile ? 0xffffu : (1u << left) - 1;
        if ((pages & 3u) != 3u) {
          if ((pages & 1u) == 0) there &= 0xff00u;
          if ((pages & 2u) == 0) there &= 0x00ffu;
        }
        uint64_t* const bar = &full[warp][slot_in];
        if (lane == 0) tc::mbar_expect_tx(bar, S::kStageBytes);
        __syncwarp();
        if (lane < order.boxes) {
          // A box that holds no key lies past the last page: zeros.
          const int p = page >= 0 ? page : static_cast<int>(a.pages);
          unsigned char* dst = ring + slot_in * S::kStageBytes + lane * 1024;
#pragma unroll 1
          for (int c = 0; c < order.copies; ++c, dst += 2048) {
            tc::tma_load_5d(dst, &k_map, 64 * c, inside, 0, batch.kv_head, p, bar);
            tc::tma_load_5d(dst + S::kKeyBytes, &v_map, 64 * c, inside, 0, batch.kv_head, p, bar);
          }
        }
      } else {
        const int64_t place =
            page < 0    ? -1
            : lane < 16 ? page * a.k_page + inside * a.k_token + batch.kv_head * a.k_head
                        : page * a.v_page + inside * a.v_token + batch.kv_head * a.v_head;
        there = pages & 0xffffu;
        // Eight lanes copy 128 bytes of one row.
        const int piece = lane & 7;
        const uint32_t dst = ring_address + slot_in * S::kStageBytes;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const int row = 4 * (s & 3) + (lane >> 3);
          const int64_t at = __shfl_sync(kFullMask, place, (s < 4 ? 0 : 16) + row);
          const T* const src =
              static_cast<const T*>(s < 4 ? a.k : a.v) + (at >= 0 ? at : 0) + 8 * piece;
          const uint32_t to = dst + row * 128 + (piece ^ (row & 7)) * 16;
#pragma unroll
          for (int c = 0; c < kDim / 64; ++c)
            copy16(to + (s < 4 ? 0 : S::kKeyBytes) + c * 2048, src + 64 * c,
                   at >= 0 && 64 * c + 8 * piece < a.head_dim);
        }
      }
      if (++slot_in == kStages) slot_in = 0;
    }
    if constexpr (!kTma) copy_commit();
    return there;
  };

  // Q in the order of the key pieces: words 0, 1 of piece j are the first
  // instruction's two k pairs, words 2, 3 the second's.  The next segment's is
  // loaded during this one, where registers allow.
  constexpr bool kQueryAhead = kDim * kRows <= 1024;
  using Query = uint4[kDim / 32][kHalves];
  Query qa, q_next;
  const auto load_query = [&](Query& x, int sequence, int unit) {
    const PagedUnit u = paged_unit<kRows>(a, unit);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const T* src = q + sequence * a.q_batch + (u.first_head + row) * a.q_head;
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) {
        const int d = 64 * (j / 2) + 16 * t + 8 * (j & 1);
        x[j][h] = row < u.rows && d < a.head_dim ? ld_ro(reinterpret_cast<const uint4*>(src + d))
                                                 : make_uint4(0, 0, 0, 0);
      }
    }
  };
  const auto load_next_query = [&]() {
    const bool same = out.unit + 1 < units;
    if (same || out.sequence + 1 < a.batch)
      load_query(q_next, same ? out.sequence : out.sequence + 1, same ? out.unit + 1 : 0);
  };
  float o[kDim / 8][4];
  float m[kHalves], l[kHalves];  // l over this lane's keys only
  const auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) m[h] = -INFINITY, l[h] = 0.0f;
  };
  clear();
  int begin = out.tile;  // of the segment
  if (to_read > 0) {
    load_query(qa, out.sequence, out.unit);
    if constexpr (kQueryAhead) load_next_query();
  }

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

    // Four chains of dependent instructions instead of two.
    float s[2][4] = {}, s_odd[2][4] = {};
#pragma unroll
    for (int j = 0; j < kDim / 32; ++j)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint4 b = ld_shared(stage + (k_piece ^ (j & 1) * 16) + (j / 2) * 2048 + n * 1024);
        Mma<T>::run(s[n], qa[j][0].x, kHalves == 2 ? qa[j][kHalves - 1].x : 0u, qa[j][0].y,
                    kHalves == 2 ? qa[j][kHalves - 1].y : 0u, b.x, b.y);
        Mma<T>::run(s_odd[n], qa[j][0].z, kHalves == 2 ? qa[j][kHalves - 1].z : 0u, qa[j][0].w,
                    kHalves == 2 ? qa[j][kHalves - 1].w : 0u, b.z, b.w);
      }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 2 * kHalves; ++x) s[n][x] = (s[n][x] + s_odd[n][x]) * a.scale_log2;
    const uint32_t seen = there[0];
    if (seen != 0xffffu) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < 2 * kHalves; ++x)
          if ((seen >> (8 * n + 2 * t + (x & 1)) & 1u) == 0) s[n][x] = -INFINITY;
    }

    float m_new[kHalves];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
      m_new[h] = fmaxf(m[h], top);
      moved |= m_new[h] != m[h];
    }
    float base[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      base[h] = m_new[h] == -INFINITY ? 0.0f : m_new[h];  // no key so far: all weights 0
    if (__any_sync(kFullMask, moved)) {
      float alpha[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        alpha[h] = paged_exp2(m[h] - base[h]);
        l[h] *= alpha[h];
        m[h] = m_new[h];
      }
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][x] *= alpha[kHalves == 2 ? x >> 1 : 0];
    }
    uint32_t p[2][kHalves], rest[2][kHalves];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const float x = paged_exp2(s[n][2 * h] - base[h]);
        const float y = paged_exp2(s[n][2 * h + 1] - base[h]);
        l[h] += x + y;
        p[n][h] = Mma<T>::split(x, y, &rest[n][h]);
      }
#pragma unroll
    for (int c = 0; c < kDim / 64; ++c) {
      uint4 v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)  // keys 2t, 2t + 1, 2t + 8, 2t + 9
        v[x] = ld_shared(stage + (x & 1 ? (v_piece ^ 16) + 128 : v_piece) + c * 2048 +
                         (x >> 1) * 1024);
      if (seen != 0xffffu) {  // what lies behind the length is not a value
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if ((seen >> (2 * t + (x & 1) + 8 * (x >> 1)) & 1u) == 0) v[x] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t b0, b1;
        if (e & 1) {
          b0 = pair_halves<true>(word(v[0], e / 2), word(v[1], e / 2));
          b1 = pair_halves<true>(word(v[2], e / 2), word(v[3], e / 2));
        } else {
          b0 = pair_halves<false>(word(v[0], e / 2), word(v[1], e / 2));
          b1 = pair_halves<false>(word(v[2], e / 2), word(v[3], e / 2));
        }
        if constexpr (kHalves == 1) {
          Mma<T>::run(o[8 * c + e], p[0][0], rest[0][0], p[1][0], rest[1][0], b0, b1);
        } else {
          Mma<T>::run(o[8 * c + e], p[0][0], p[0][kHalves - 1], p[1][0], p[1][kHalves - 1], b0,
                      b1);
          Mma<T>::run(o[8 * c + e], rest[0][0], rest[0][kHalves - 1], rest[1][0],
                      rest[1][kHalves - 1], b0, b1);
        }
      }
    }

    --to_read;
    if (out.tile + 1 < out.tiles && to_read > 0) {
      ++out.tile;
      continue;
    }

    // The segment ends.
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
      l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
    }
    if constexpr (kHalves == 1) {
      // An infinite value times a rest of zero is no number; the first part of
      // the weight alone gives the infinity.
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (o[n][2 + x] == o[n][2 + x]) o[n][x] += o[n][2 + x];
    }
    const PagedUnit unit = paged_unit<kRows>(a, out.unit);
    const bool whole = begin == 0 && out.tile + 1 == out.tiles;
    // A part goes to the ring, which is empty, when the warp is done, else out
    // of its way.
    const bool spilled = to_read > 0;
    const int kind = begin == 0 ? kTail : kHead;
    float* const part = spilled ? a.spill + range * a.row_cap * a.head_dim
                                : reinterpret_cast<float*>(ring);
    const int pitch = spilled ? a.head_dim : S::kPitch;
    if constexpr (!kTma) {
      if (!whole) copy_wait<0>();
    }
    __syncwarp();  // every lane has read its last stage
    // The lane's rows are g + 8h; of piece c it holds columns 8 (2t + x) + e in
    // o[8c + e][2h + x].
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      if (row >= unit.rows) continue;
      T* const dst =
          static_cast<T*>(a.out) +
          (static_cast<int64_t>(out.sequence) * a.heads + unit.first_head + row) * a.head_dim;
      const float f = !whole ? 1.0f : out.length == 0 ? 0.0f : __fdividef(1.0f, l[h]);
#pragma unroll
      for (int c = 0; c < kDim / 64; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int d = 64 * c + 8 * (2 * t + x);
          if (d >= a.head_dim) continue;
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = o[8 * c + e][2 * h + x] * f;
          if (whole) {
            alignas(16) T z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) st_out(&z[e], y[e]);
            *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(z);
          } else {
            float4* const to = reinterpret_cast<float4*>(part + row * pitch + d);
            to[0] = make_float4(y[0], y[1], y[2], y[3]);
            to[1] = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      if (!whole && t == 0) {
        parts.m[warp][kind][row] = m[h];
        parts.l[warp][kind][row] = l[h];
      }
    }
    if (!whole && lane == 0)
      parts.records[warp][kind] = PartRecord{out.sequence, out.unit,     out.tiles, begin,
                                             out.tile + 1, opens && kind == kHead, spilled};
    if (to_read > 0) {
      advance(out);
      begin = 0;
      clear();
      if constexpr (kQueryAhead) {
#pragma unroll
        for (int j = 0; j < kDim / 32; ++j)
#pragma unroll
          for (int h = 0; h < kHalves; ++h) qa[j][h] = q_next[j][h];
        load_next_query();
      } else {
        load_query(qa, out.sequence, out.unit);
      }
    }
  }
  if (reported != 0) watchdog_trip(a.watchdog, reported);
  __syncthreads();
  paged_merge<T, kWarps, kRows, S::kRingBytes / 4, S::kPitch, 4>(
      a, parts, reinterpret_cast<const float*>(rings));
}

// Encodes a cache for the TMA unit; false when its layout does not allow it.
template <typename T>
bool cache_map(CUtensorMap* map, const PagedArgs& a, const void* base, int64_t page, int64_t token,
               int64_t head, const MapOrder& order) {
  const uint64_t page_size = a.page_size.divisor;
  const uint64_t pieces = order.copies == 1 ? (a.head_dim + 63) / 64 : 1;
  const uint64_t extent[5] = {static_cast<uint64_t>(order.copies == 1 && a.head_dim > 64 ? 64 : a.head_dim),
                        page_size, pieces, static_cast<uint64_t>(a.kv_heads),
                        static_cast<uint64_t>(a.pages)};
  int64_t stride[4] = {token, 64, head, page};
  const uint32_t box[5] = {64, static_cast<uint32_t>(kTile / order.boxes), static_cast<uint32_t>(pieces), 1,
                     1};
  uint64_t bytes[4];
  for (int i = 0; i < 4; ++i) {
    // A dimension of one element may come with any stride.
    if (extent[i + 1] == 1) stride[i] = 8;
    if (stride[i] <= 0 || stride[i] >= (int64_t{1} << 39)) return false;
    bytes[i] = static_cast<uint64_t>(stride[i]) * sizeof(T);
  }
  const CUtensorMapDataType type = sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return encode_tmap(map, type, 5, base, extent, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B) ==
         cudaSuccess;
}

template <typename T, int kDim, int kRows, bool kTma, int kWarps, int kStages>
int launch_mma(PagedArgs a, const CUtensorMap& k_map, const CUtensorMap& v_map,
               const MapOrder& order, cudaStream_t stream) {
  constexpr auto kernel = paged_mma_kernel<T, kDim, kRows, kTma, kWarps, kStages>;
  constexpr size_t kShared = Shape<T, kDim, kRows, kWarps, kStages>::kShared;
  const int grid = paged_grid(a, sm_count(), kTile, kWarps, kRows);
  paged_scratch(&a, grid, kWarps, kRows);
  cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(kShared));
  if (error != cudaSuccess) return error;
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
    error = launch_join<T, kTile, kWarps, kRows>(a, grid, stream);
  return error != cudaSuccess ? error : cudaGetLastError();
}

template <typename T, int kRows, bool kTma>
int pick_dim(const PagedArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map,
             const MapOrder& order, cudaStream_t stream) {
  // About 192 KB of rings a CTA, one CTA a SM.
  if (a.head_dim <= 64) return launch_mma<T, 64, kRows, kTma, 8, 3>(a, k_map, v_map, order, stream);
  if (a.head_dim <= 128)
    return launch_mma<T, 128, kRows, kTma, 8, 2>(a, k_map, v_map, order, stream);
  if (a.head_dim <= 192)
    return launch_mma<T, 192, kRows, kTma, 4, 3>(a, k_map, v_map, order, stream);
  return launch_mma<T, 256, kRows, kTma, 4, 2>(a, k_map, v_map, order, stream);
}

}  // namespace

template <typename T>
int paged_attention_mma(PagedArgs a, cudaStream_t stream) {
  if (a.pages > 0x7fffffff) a.pages = 0x7fffffff;  // as far as block-table entries reach
  CUtensorMap k_map = {}, v_map = {};
  MapOrder order = {a.page_size.divisor % kTile == 0 ? 1 : 2, (a.head_dim + 63) / 64};
  if (order.boxes == 1 && a.head_dim % 64 == 0) order.copies = 1;
  const bool tma =
      a.page_size.divisor % 8 == 0 &&
      cache_map<T>(&k_map, a, a.k, a.k_page, a.k_token, a.k_head, order) &&
      cache_map<T>(&v_map, a, a.v, a.v_page, a.v_token, a.v_head, order);
  if (tma)
    return a.group <= 8 ? pick_dim<T, 8, true>(a, k_map, v_map, order, stream)
                        : pick_dim<T, 16, true>(a, k_map, v_map, order, stream);
  return a.group <= 8 ? pick_dim<T, 8, false>(a, k_map, v_map, order, stream)
                      : pick_dim<T, 16, false>(a, k_map, v_map, order, stream);
}

template int paged_attention_mma<__half>(PagedArgs, cudaStream_t);
template int paged_attention_mma<__nv_bfloat16>(PagedArgs, cudaStream_t);

}  // namespace opl
