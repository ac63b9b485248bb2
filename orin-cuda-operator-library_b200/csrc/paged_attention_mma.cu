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
#include <utility>

#include "paged_attention.cuh"
#include "tc_common.cuh"
#include "tmap.cuh"

namespace opl {

namespace {

constexpr int kTile = 16;
// Block-table entries are loaded this many steps before their copies.
constexpr int kAhead = 2;

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

// How the tensor maps of the caches are laid out.
struct MapOrder {
  int token_first;  // dimensions (head_dim, token, head, page), else head before token
  int boxes;        // of a tile: one of 16 tokens, or two of 8
};

// Copies are made by the TMA unit, or by the lanes (kTma false).
template <typename T, int kDim, int kRows, bool kTma, int kWarps, int kStages, int kLeast>
__global__ void __launch_bounds__(32 * kWarps, 1)
    paged_mma_kernel(const PagedArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map, const MapOrder order, int row_cap) {
  using S = Shape<T, kDim, kRows, kWarps, kStages>;
  constexpr int kThreads = 32 * kWarps;
  constexpr int kHalves = kRows / 8;  // row groups of the S accumulator in use
  extern __shared__ unsigned char shared[];
  __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];
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
  pdl_begin();

  const T* q = static_cast<const T*>(a.q);
  const int page_size = static_cast<int>(a.page_size.divisor);
  // The barriers are also set up before the first copy by this search's
  // __syncthreads.
  const PagedStart start = paged_start<kThreads, kTile, kLeast>(
      a, gridDim.x, [](long long total, int ctas) -> long long {
        return static_cast<int>(blockIdx.x) < ctas ? range_begin(total, ctas, blockIdx.x) : -1;
      });
  if (static_cast<int>(blockIdx.x) >= start.ctas) return;
  int64_t w = range_begin(start.total, start.ctas, blockIdx.x);
  const int64_t limit = range_begin(start.total, start.ctas, blockIdx.x + 1);
  int sequence = start.sequence;
  int64_t before = start.before;
  int reported = 0;
  int slot_in = 0, slot_out = 0;  // ring stages being filled and read
  uint32_t parity = 0;            // of the stage being read
  bool dead = false;              // a wait gave up; the warp copies no more

  // Where this lane's pieces lie in a stage (see the layout above).
  const uint32_t k_piece = g * 128 + (2 * t ^ g) * 16;
  const uint32_t v_piece = S::kKeyBytes + 2 * t * 128 + (g ^ 2 * t) * 16;
  const uint32_t ring_address = tc::smem_u32(ring);

  while (w < limit) {
    const int raw_length = ld_int(a.seq_lens + sequence);
    const int length = readable_length(raw_length, a.max_pages, page_size);
    if (length != raw_length) reported = kBadLength;
    const int tiles = key_tiles(length, kTile);
    if (w >= (before + tiles) * a.units()) {
      before += tiles;
      ++sequence;
      continue;
    }
    const Segment segment = segment_at(w, limit, before, tiles, a.units());
    w += segment.end - segment.begin;
    const PagedUnit unit = paged_unit<kRows>(a, segment.unit);
    const int* table = a.block_table + sequence * a.table_row;
    const int first = segment.begin + warp;
    const int count = !dead && first < segment.end ? (segment.end - first - 1) / kWarps + 1 : 0;

    // The key that this lane places in tile i: with the TMA unit the first of
    // a box of 16 or 8 (even and odd lanes: first and second half of the
    // tile), else lanes 0-15 a key each and lanes 16-31 their values.  Its
    // block-table entry is loaded some steps before it is used.
    const auto key_of = [&](int i) {
      return (first + i * kWarps) * kTile + (kTma ? 8 * (lane & 1) : lane & 15);
    };
    const auto fetch = [&](int i) {
      const int key = key_of(i);
      return i < count && key < length ? ld_int(table + fast_div(key, a.page_size)) : 0;
    };
    // Copies tile i into the next stage; bit j of the result: key j is there.
    const auto issue = [&](int i, int page) -> uint32_t {
      uint32_t there = 0;
      if (i < count) {
        const int key = key_of(i);
        const bool known = key < length;
        const bool ok = known && cache_page(page, a.pages);
        if (known && !ok) reported = kBadPage;
        const int inside = key - static_cast<int>(fast_div(key, a.page_size)) * page_size;
        if constexpr (kTma) {
          const uint32_t halves = __ballot_sync(kFullMask, ok) & 3u;
          const int left = length - (first + i * kWarps) * kTile;
          there = left >= kTile ? 0xffffu : (1u << left) - 1;
          if ((halves & 1u) == 0) there &= 0xff00u;
          if ((halves & 2u) == 0) there &= 0x00ffu;
          uint64_t* const bar = &full[warp][slot_in];
          if (lane == 0) tc::mbar_expect_tx(bar, S::kStageBytes);
          __syncwarp();
          if (lane < order.boxes) {
            // A box that holds no key lies past the last page: zeros.
            const int p = ok ? page : static_cast<int>(a.pages);
            const int y = order.token_first ? inside : unit.kv_head;
            const int z = order.token_first ? unit.kv_head : inside;
            unsigned char* dst = ring + slot_in * S::kStageBytes + lane * 1024;
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c)
              tc::tma_load_4d(dst + c * 2048, &k_map, 64 * c, y, z, p, bar);
#pragma unroll
            for (int c = 0; c < kDim / 64; ++c)
              tc::tma_load_4d(dst + S::kKeyBytes + c * 2048, &v_map, 64 * c, y, z, p, bar);
          }
        } else {
          const int64_t place = !ok ? -1
                                : lane < 16
                                    ? page * a.k_page + inside * a.k_token + unit.kv_head * a.k_head
                                    : page * a.v_page + inside * a.v_token + unit.kv_head * a.v_head;
          there = __ballot_sync(kFullMask, ok) & 0xffffu;
          // Eight lanes copy 128 bytes of one row.
          const int piece = lane & 7;
          uint32_t dst = ring_address + slot_in * S::kStageBytes;
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

    uint32_t there[kStages];
    int pages[kStages - 1 + kAhead];
#pragma unroll
    for (int i = 0; i < kStages - 1 + kAhead; ++i) pages[i] = fetch(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) there[i] = issue(i, pages[i]);

    // Q in the order of the key pieces: words 0, 1 of piece j are the first
    // instruction's two k pairs, words 2, 3 the second's.
    uint4 qa[kDim / 32][kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const T* src = q + sequence * a.q_batch + (unit.first_head + row) * a.q_head;
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) {
        const int d = 64 * (j / 2) + 16 * t + 8 * (j & 1);
        qa[j][h] = row < unit.rows && d < a.head_dim ? ld_ro(reinterpret_cast<const uint4*>(src + d))
                                                     : make_uint4(0, 0, 0, 0);
      }
    }
    float o[kDim / 8][4];
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[kHalves], l[kHalves];  // l over this lane's keys only
#pragma unroll
    for (int h = 0; h < kHalves; ++h) m[h] = -INFINITY, l[h] = 0.0f;

    for (int i = 0; i < count; ++i) {
      const int later_page = fetch(i + kStages - 1 + kAhead);
      __syncwarp();  // every lane has read the stage that is filled next
      there[kStages - 1] = issue(i + kStages - 1, pages[kStages - 1]);
#pragma unroll
      for (int x = kStages - 1; x < kStages - 2 + kAhead; ++x) pages[x] = pages[x + 1];
      pages[kStages - 2 + kAhead] = later_page;
      if constexpr (kTma) {
        if (!tc::mbar_wait_warp(&full[warp][slot_out], parity, &abort_wait, a.watchdog,
                                tc::kWatchdogPaged)) {
          // Give the other copies in flight the same time to land, then leave
          // the segment; the output is not valid and the watchdog says so.
          for (int x = 1; x < kStages && i + x < count; ++x) {
            const int slot = (slot_out + x) % kStages;
            volatile int alone = 0;
            tc::mbar_wait(&full[warp][slot], slot < slot_out ? parity ^ 1u : parity, &alone,
                          a.watchdog, tc::kWatchdogPaged);
          }
          dead = true;
          break;
        }
      } else {
        copy_wait<kStages - 1>();
        __syncwarp();  // what the other lanes copied
      }
      const uint32_t stage = ring_address + slot_out * S::kStageBytes;
      if (++slot_out == kStages) slot_out = 0, parity ^= 1u;

      float s[2][4] = {};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < kDim / 32; ++j) {
          const uint4 b = ld_shared(stage + (k_piece ^ (j & 1) * 16) + (j / 2) * 2048 + n * 1024);
          Mma<T>::run(s[n], qa[j][0].x, kHalves == 2 ? qa[j][kHalves - 1].x : 0u, qa[j][0].y,
                      kHalves == 2 ? qa[j][kHalves - 1].y : 0u, b.x, b.y);
          Mma<T>::run(s[n], qa[j][0].z, kHalves == 2 ? qa[j][kHalves - 1].z : 0u, qa[j][0].w,
                      kHalves == 2 ? qa[j][kHalves - 1].w : 0u, b.z, b.w);
        }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < 2 * kHalves; ++x) s[n][x] *= a.scale_log2;
      const uint32_t seen = there[0];
      if (seen != 0xffffu) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 2 * kHalves; ++x)
            if ((seen >> (8 * n + 2 * t + (x & 1)) & 1u) == 0) s[n][x] = -INFINITY;
      }
#pragma unroll
      for (int x = 0; x + 1 < kStages; ++x) there[x] = there[x + 1];

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
    }
    if constexpr (!kTma) copy_wait<0>();

    // Merge the warps, each through its own (now empty) ring.
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
      l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
      if (t == 0) {
        merge_m[warp][g + 8 * h] = m[h];
        merge_l[warp][g + 8 * h] = l[h];
      }
    }
    __syncwarp();  // the ring is written across lanes from here
    float* const merge_o = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int c = 0; c < kDim / 64; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x)  // columns 8 (2t + x) + e of the piece
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            float4 out;
            float* const f = &out.x;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float (&acc)[4] = o[8 * c + e + y];
              if constexpr (kHalves == 1) {
                // An infinite value times a rest of zero is no number; the
                // first part of the weight alone gives the infinity.
                f[y] = acc[2 + x] == acc[2 + x] ? acc[x] + acc[2 + x] : acc[x];
              } else {
                f[y] = acc[2 * h + x];
              }
            }
            *reinterpret_cast<float4*>(merge_o + (g + 8 * h) * S::kPitch + 64 * c + 8 * (2 * t + x) +
                                       e) = out;
          }
    __syncthreads();
    const int slot = 2 * blockIdx.x + segment.slot();
    for (int i = threadIdx.x; i < unit.rows * a.head_dim; i += kThreads) {
      const int r = i / a.head_dim, d = i - r * a.head_dim;
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) top = fmaxf(top, merge_m[x][r]);
      const float base_m = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, out = 0.0f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float f = paged_exp2(merge_m[x][r] - base_m);
        sum = fmaf(f, merge_l[x][r], sum);
        out = fmaf(f, reinterpret_cast<const float*>(rings + x * S::kRingBytes)[r * S::kPitch + d],
                   out);
      }
      if (segment.whole()) {
        st_out(static_cast<T*>(a.out) +
                   (static_cast<int64_t>(sequence) * a.heads + unit.first_head + r) * a.head_dim + d,
               length == 0 ? 0.0f : out / sum);
      } else {
        const int64_t row = static_cast<int64_t>(slot) * row_cap + r;
        a.partial[row * a.head_dim + d] = out;
        if (d == 0) a.partial_ml[row] = make_float2(top, sum);
      }
    }
    // The rings go back to the TMA unit.
    if constexpr (kTma) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  if (reported != 0) watchdog_trip(a.watchdog, reported);
}

// Encodes a cache for the TMA unit; false when its layout does not allow it.
template <typename T>
bool cache_map(CUtensorMap* map, const PagedArgs& a, const void* base, int64_t page, int64_t token,
               int64_t head, const MapOrder& order) {
  const uint64_t page_size = a.page_size.divisor;
  uint64_t extent[4] = {static_cast<uint64_t>(a.head_dim), page_size,
                        static_cast<uint64_t>(a.kv_heads), static_cast<uint64_t>(a.pages)};
  int64_t stride[3] = {token, head, page};
  uint32_t box[4] = {64, static_cast<uint32_t>(kTile / order.boxes), 1, 1};
  if (!order.token_first) {
    std::swap(extent[1], extent[2]);
    std::swap(stride[0], stride[1]);
    std::swap(box[1], box[2]);
  }
  uint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    // A dimension of one element may come with any stride.
    if (extent[i + 1] == 1) stride[i] = 8;
    if (stride[i] <= 0 || stride[i] >= (int64_t{1} << 39)) return false;
    bytes[i] = static_cast<uint64_t>(stride[i]) * sizeof(T);
  }
  const CUtensorMapDataType type = sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return encode_tmap(map, type, 4, base, extent, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B) ==
         cudaSuccess;
}

template <typename T, int kDim, int kRows, bool kTma, int kWarps, int kStages>
int launch_mma(PagedArgs a, const CUtensorMap& k_map, const CUtensorMap& v_map,
               const MapOrder& order, cudaStream_t stream) {
  constexpr int kLeast = kWarps;
  constexpr auto kernel = paged_mma_kernel<T, kDim, kRows, kTma, kWarps, kStages, kLeast>;
  constexpr size_t kShared = Shape<T, kDim, kRows, kWarps, kStages>::kShared;
  a.parts = (a.group + kRows - 1) / kRows;
  const int row_cap = a.group < kRows ? a.group : kRows;
  const int grid = paged_grid(a, sm_count(), kTile, kLeast, kRows);
  a.partial_ml = reinterpret_cast<float2*>(a.partial + static_cast<int64_t>(grid) * 2 * row_cap *
                                                           a.head_dim);
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
  error = cudaLaunchKernelEx(&config, kernel, a, k_map, v_map, order, row_cap);
  if (error == cudaSuccess && grid > 1)
    error = launch_join<T, kTile, kLeast, kRows>(a, grid, row_cap, stream);
  return error != cudaSuccess ? error : cudaGetLastError();
}

template <typename T, int kRows, bool kTma>
int pick_dim(const PagedArgs& a, const CUtensorMap& k_map, const CUtensorMap& v_map,
             const MapOrder& order, cudaStream_t stream) {
  // About 192 KB of rings a CTA, one CTA a SM.
  if (a.head_dim <= 64) return launch_mma<T, 64, kRows, kTma, 8, 6>(a, k_map, v_map, order, stream);
  if (a.head_dim <= 128)
    return launch_mma<T, 128, kRows, kTma, 8, 3>(a, k_map, v_map, order, stream);
  if (a.head_dim <= 192)
    return launch_mma<T, 192, kRows, kTma, 4, 4>(a, k_map, v_map, order, stream);
  return launch_mma<T, 256, kRows, kTma, 4, 3>(a, k_map, v_map, order, stream);
}

}  // namespace

template <typename T>
int paged_attention_mma(PagedArgs a, cudaStream_t stream) {
  if (a.pages > 0x7fffffff) a.pages = 0x7fffffff;  // as far as block-table entries reach
  CUtensorMap k_map = {}, v_map = {};
  MapOrder order = {a.k_token < a.k_head ? 1 : 0, a.page_size.divisor % kTile == 0 ? 1 : 2};
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
