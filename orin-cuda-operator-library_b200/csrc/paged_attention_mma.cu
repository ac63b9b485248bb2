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
// One warp owns 16 keys at a time and never waits for another one:
//
// * Every lane copies by cp.async exactly the 16-byte pieces that it will
//   itself use as operands, into a ring of its own, kStages deep.  No barrier
//   guards the ring, each piece is read back by a conflict-free 128-bit load,
//   and 8 warps x 3 stages keep 192 KB (head size 128) in flight per SM; about
//   50 KB cover the latency at the full rate.
// * That works because a contraction may run over its index in any order.
//   S = Q K^T: lane (g, t) of an m16n8k16 B operand holds row g (key g), any
//   8 consecutive elements of the head per two instructions; Q is loaded in
//   the same order.  O = P V: the operand pairs two keys of one column, so the
//   lane loads 8 consecutive columns of keys 2t, 2t+1, 2t+8, 2t+9 -- the keys
//   whose weights the S accumulator left in this lane -- and one byte permute
//   a register pairs them; instruction e of 8 then computes columns 8n + e of
//   the head, which lands 8 consecutive columns of a row in one lane.
// * The weights enter P V as the sum of two 16-bit values, so that their
//   rounding (2^-9 in BF16, as much as the result's own) does not show.  With
//   up to 8 query heads a unit the second value rides in the 8 rows of the
//   operand that are otherwise empty.
//
// Running maximum, sum and output are FP32 in registers; the warps of a CTA
// merge at the end of a segment, and cut units are joined by a second launch.
#include "paged_attention.cuh"

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
  static constexpr int kKeyChunks = 2 * (kDim / 32);    // 16-byte pieces a lane and tile
  static constexpr int kValueChunks = 4 * (kDim / 64);
  static constexpr int kStageBytes = (kKeyChunks + kValueChunks) * 512;
  static constexpr int kRingBytes = kStages * kStageBytes;  // of a warp
  static constexpr int kPitch = kDim + 4;  // of a merged row, in floats
  static constexpr size_t kShared = static_cast<size_t>(kWarps) * kRingBytes;
  static_assert(kRows * kPitch * 4 <= kRingBytes, "a warp merges through its own ring");
  static_assert(kShared <= 220 * 1024, "beside the static arrays");
};

template <typename T, int kDim, int kRows, int kWarps, int kStages, int kLeast>
__global__ void __launch_bounds__(32 * kWarps, 1) paged_mma_kernel(const PagedArgs a, int row_cap) {
  using S = Shape<T, kDim, kRows, kWarps, kStages>;
  constexpr int kThreads = 32 * kWarps;
  constexpr int kHalves = kRows / 8;  // row groups of the S accumulator in use
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float merge_m[kWarps][kRows], merge_l[kWarps][kRows];
  pdl_begin();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t my_ring =
      static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * S::kRingBytes + lane * 16;
  const T* q = static_cast<const T*>(a.q);
  const T* keys = static_cast<const T*>(a.k);
  const T* values = static_cast<const T*>(a.v);
  const int page_size = static_cast<int>(a.page_size.divisor);
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
    const T* k_head = keys + unit.kv_head * a.k_head;
    const T* v_head = values + unit.kv_head * a.v_head;
    const int first = segment.begin + warp;
    const int count = first < segment.end ? (segment.end - first - 1) / kWarps + 1 : 0;

    // Lanes 0-15 place the keys of a tile, lanes 16-31 its values; the
    // block-table entry is loaded a step before it is used.
    const auto fetch = [&](int i) {
      const int key = (first + i * kWarps) * kTile + (lane & 15);
      return i < count && key < length ? ld_int(table + fast_div(key, a.page_size)) : 0;
    };
    // Copies tile i into its stage; bit j of the result: key j is there.
    const auto issue = [&](int i, int page) -> uint32_t {
      uint32_t there = 0;
      if (i < count) {
        const int key = (first + i * kWarps) * kTile + (lane & 15);
        int64_t place = -1;
        if (key < length) {
          if (cache_page(page, a.pages)) {
            const int inside =
                key - static_cast<int>(fast_div(key, a.page_size)) * page_size;
            place = lane < 16 ? page * a.k_page + inside * a.k_token
                              : page * a.v_page + inside * a.v_token;
          } else {
            reported = kBadPage;
          }
        }
        there = __ballot_sync(kFullMask, place >= 0) & 0xffffu;
        uint32_t dst = my_ring + (i % kStages) * S::kStageBytes;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int64_t at = __shfl_sync(kFullMask, place, 8 * n + g);
#pragma unroll
          for (int j = 0; j < kDim / 32; ++j, dst += 512) {
            const int d = 32 * j + 8 * t;
            const bool ok = at >= 0 && d < a.head_dim;
            copy16(dst, ok ? k_head + at + d : keys, ok);
          }
        }
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const int64_t at =
              __shfl_sync(kFullMask, place, 16 + 2 * t + (i4 & 1) + 8 * (i4 >> 1));
#pragma unroll
          for (int c = 0; c < kDim / 64; ++c, dst += 512) {
            const int d = 64 * c + 8 * g;
            const bool ok = at >= 0 && d < a.head_dim;
            copy16(dst, ok ? v_head + at + d : values, ok);
          }
        }
      }
      copy_commit();
      return there;
    };

    uint32_t there[kStages];
    int pages[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) pages[i] = fetch(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) there[i] = issue(i, pages[i]);
    int next_page = pages[kStages - 1];

    // Q in the order of the key pieces: words 0, 1 of piece j are the first
    // instruction's two k pairs, words 2, 3 the second's.
    uint4 qa[kDim / 32][kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const T* src = q + sequence * a.q_batch + (unit.first_head + row) * a.q_head;
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) {
        const int d = 32 * j + 8 * t;
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
      const int later_page = fetch(i + kStages);
      there[kStages - 1] = issue(i + kStages - 1, next_page);
      next_page = later_page;
      copy_wait<kStages - 1>();
      uint32_t src = my_ring + (i % kStages) * S::kStageBytes;

      float s[2][4] = {};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < kDim / 32; ++j, src += 512) {
          const uint4 b = ld_shared(src);
          Mma<T>::run(s[n], qa[j][0].x, kHalves == 2 ? qa[j][kHalves - 1].x : 0u, qa[j][0].y,
                      kHalves == 2 ? qa[j][kHalves - 1].y : 0u, b.x, b.y);
          Mma<T>::run(s[n], qa[j][0].z, kHalves == 2 ? qa[j][kHalves - 1].z : 0u, qa[j][0].w,
                      kHalves == 2 ? qa[j][kHalves - 1].w : 0u, b.z, b.w);
        }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int x = 0; x < 2 * kHalves; ++x) s[n][x] *= a.scale_log2;
      if (there[0] != 0xffffu) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 2 * kHalves; ++x)
            if ((there[0] >> (8 * n + 2 * t + (x & 1)) & 1u) == 0) s[n][x] = -INFINITY;
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
        for (int i4 = 0; i4 < 4; ++i4) v[i4] = ld_shared(src + (i4 * (kDim / 64) + c) * 512);
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
    copy_wait<0>();

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
    float* const merge_o = reinterpret_cast<float*>(ring + warp * S::kRingBytes);
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
        out = fmaf(f, reinterpret_cast<const float*>(ring + x * S::kRingBytes)[r * S::kPitch + d],
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
    __syncthreads();
  }
  if (reported != 0) watchdog_trip(a.watchdog, reported);
}

template <typename T, int kDim, int kRows, int kWarps, int kStages>
int launch_mma(PagedArgs a, cudaStream_t stream) {
  constexpr int kLeast = kWarps;
  constexpr auto kernel = paged_mma_kernel<T, kDim, kRows, kWarps, kStages, kLeast>;
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
  error = cudaLaunchKernelEx(&config, kernel, a, row_cap);
  if (error == cudaSuccess && grid > 1)
    error = launch_join<T, kTile, kLeast, kRows>(a, grid, row_cap, stream);
  return error != cudaSuccess ? error : cudaGetLastError();
}

template <typename T, int kRows>
int pick_dim(const PagedArgs& a, cudaStream_t stream) {
  // About 192 KB of rings a CTA, one CTA a SM.
  if (a.head_dim <= 64) return launch_mma<T, 64, kRows, 8, 6>(a, stream);
  if (a.head_dim <= 128) return launch_mma<T, 128, kRows, 8, 3>(a, stream);
  if (a.head_dim <= 192) return launch_mma<T, 192, kRows, 4, 4>(a, stream);
  return launch_mma<T, 256, kRows, 4, 3>(a, stream);
}

}  // namespace

template <typename T>
int paged_attention_mma(PagedArgs a, cudaStream_t stream) {
  return a.group <= 8 ? pick_dim<T, 8>(a, stream) : pick_dim<T, 16>(a, stream);
}

template int paged_attention_mma<__half>(PagedArgs, cudaStream_t);
template int paged_attention_mma<__nv_bfloat16>(PagedArgs, cudaStream_t);

}  // namespace opl
