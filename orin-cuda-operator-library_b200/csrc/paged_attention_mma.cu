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
// The tiles come through paged_stream.cuh, 16 keys at a time.
//
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
// * The weights enter P V as the sum of two 16-bit values: one alone would
//   round by 2^-8 in BF16, as much as the result itself; two leave 2^-16 of a
//   weight, and 2^-22 in FP16.  FP16 also ends at steps of 2^-24, so its weights
//   (and their sum: the factor cancels) are held times 2^15: half a step is
//   2^-40 of the largest weight, not 2^-25, which a long tail below one key
//   shows.  With up to 8 query heads a unit the second value rides in the 8
//   rows of the operand that are otherwise empty.
//
// Running maximum, sum and output are FP32 in registers.
#include "paged_stream.cuh"

namespace opl {

namespace {

template <typename T>
struct Mma;
template <>
struct Mma<__half> {
  static constexpr uint32_t kInfinity = 0x7c00;
  static constexpr float kWeightScale = 32768.0f;  // of weights up to 1: all below 65504
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
  static constexpr uint32_t kInfinity = 0x7f80;
  static constexpr float kWeightScale = 1.0f;
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
template <typename T_, int kDim_, int kRows_>
struct MmaPolicy {
  using T = T_;
  static constexpr int kTile = 16, kDim = kDim_, kRows = kRows_, kWarpShared = 0;
  static constexpr bool kInfiniteValues = true;  // take a second look
  static constexpr int kHalves = kRows / 8;  // row groups of the S accumulator in use
  // The next segment's queries have registers of their own where there are any.
  static constexpr bool kQueryAhead = kDim * kRows <= 1024;
  // Q in the order of the key pieces: words 0, 1 of piece j are the first
  // instruction's two k pairs, words 2, 3 the second's.
  using Query = uint4[kDim / 32][kHalves];
  Query qa, q_next;
  float o[kDim / 8][4];
  float m[kHalves], l[kHalves];  // l over this lane's keys only, times kWeightScale as o is
  int g, t;
  uint32_t k_piece, v_piece;  // where this lane's pieces lie

  __device__ __forceinline__ void init(int lane, float*) {
    g = lane >> 2, t = lane & 3;
    k_piece = g * 128 + (2 * t ^ g) * 16;
    v_piece = 2 * t * 128 + (g ^ 2 * t) * 16;
  }

  __device__ __forceinline__ void load(Query& x, const PagedArgs& a, int sequence, int index) const {
    const PagedUnit u = paged_unit<kRows>(a, index);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      const T* src =
          static_cast<const T*>(a.q) + sequence * a.q_batch + (u.first_head + row) * a.q_head;
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j) {
        const int d = 64 * (j / 2) + 16 * t + 8 * (j & 1);
        x[j][h] = row < u.rows && d < a.head_dim ? ld_ro(reinterpret_cast<const uint4*>(src + d))
                                                 : make_uint4(0, 0, 0, 0);
      }
    }
  }

  __device__ __forceinline__ void fetch_query(const PagedArgs& a, int sequence, int index) {
    if constexpr (kQueryAhead) load(q_next, a, sequence, index);
  }

  __device__ __forceinline__ void start(const PagedArgs& a, int sequence, int index) {
    if constexpr (kQueryAhead) {
#pragma unroll
      for (int j = 0; j < kDim / 32; ++j)
#pragma unroll
        for (int h = 0; h < kHalves; ++h) qa[j][h] = q_next[j][h];
    } else {
      load(qa, a, sequence, index);
    }
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) m[h] = -INFINITY, l[h] = 0.0f;
  }

  // A tile at shared addresses `keys` and `values`; bit j of `seen`: key j is
  // there.
  __device__ __forceinline__ void step(const PagedArgs& a, uint32_t keys, uint32_t values,
                                       uint32_t seen) {
    // Four chains of dependent instructions instead of two.
    float s[2][4] = {}, s_odd[2][4] = {};
#pragma unroll
    for (int j = 0; j < kDim / 32; ++j)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint4 b = ld_shared(keys + (k_piece ^ (j & 1) * 16) + (j / 2) * 2048 + n * 1024);
        Mma<T>::run(s[n], qa[j][0].x, kHalves == 2 ? qa[j][kHalves - 1].x : 0u, qa[j][0].y,
                    kHalves == 2 ? qa[j][kHalves - 1].y : 0u, b.x, b.y);
        Mma<T>::run(s_odd[n], qa[j][0].z, kHalves == 2 ? qa[j][kHalves - 1].z : 0u, qa[j][0].w,
                    kHalves == 2 ? qa[j][kHalves - 1].w : 0u, b.z, b.w);
      }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 2 * kHalves; ++x) s[n][x] = (s[n][x] + s_odd[n][x]) * a.scale_log2;
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
        const float x = paged_exp2(s[n][2 * h] - base[h]) * Mma<T>::kWeightScale;
        const float y = paged_exp2(s[n][2 * h + 1] - base[h]) * Mma<T>::kWeightScale;
        l[h] += x + y;
        p[n][h] = Mma<T>::split(x, y, &rest[n][h]);
      }
#pragma unroll
    for (int c = 0; c < kDim / 64; ++c) {
      uint4 v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)  // keys 2t, 2t + 1, 2t + 8, 2t + 9
        v[x] = ld_shared(values + (x & 1 ? (v_piece ^ 16) + 128 : v_piece) + c * 2048 +
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

  // Ends a segment: sums over the lanes that hold different keys.  True when an
  // output is not finite (see infinite_values), no key has a weight, or a score is no
  // number.
  __device__ __forceinline__ bool settle() {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
      l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
    }
    // No number once an output is not finite; the second eight rows read the same
    // values as the first.
    float odd[4] = {};
#pragma unroll
    for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if constexpr (kHalves == 1) o[n][x] += o[n][2 + x];
        odd[2 * (n & 1) + x] = fmaf(o[n][x], 0.0f, odd[2 * (n & 1) + x]);
      }
    const float any = (odd[0] + odd[1]) + (odd[2] + odd[3]);
    return __any_sync(kFullMask, any != any || !(l[0] > 0.0f) || !(l[kHalves - 1] > 0.0f));
  }

  // An infinite value times the two parts of a weight, of which the second may
  // be negative and either zero, is no number.  So the columns that read an
  // infinity or NaN among keys first .. end - 1 of the segment are written again
  // from a second look at them: store(row, column, value).  After the outputs,
  // whose registers are free then (before them: 16/1 heads of 256 33.6 us).  The
  // sums that call for it cost 1.5% of 256 short sequences, 31.0 -> 31.5 us, and
  // 4% of 16/1 heads of 256, 31.4 -> 32.7 us.  The look itself, where it is taken:
  // 314 -> 781 us for 128 sequences of up to 8191 keys, every value NaN.
  template <typename Store>
  __device__ __forceinline__ void infinite_values(const PagedArgs& a, const PagedUnit& unit,
                                                  int sequence, int first, int end,
                                                  Store store) const {
    bool sums = false;  // a row with a sum; the others are no numbers at all
#pragma unroll
    for (int h = 0; h < kHalves; ++h) sums |= g + 8 * h < unit.rows && l[h] > 0.0f;
    if (!__any_sync(kFullMask, sums)) return;
    const int* const table = a.block_table + sequence * a.table_row;
    const T* const head = static_cast<const T*>(a.v) + unit.kv_head * a.v_head;
    // Pieces of 8 columns, as in each(): all at once, but one by one for heads over
    // 128, whose kernels have no registers to spare (32.7 against 33.8 us).
    constexpr int kPieces = kDim > 128 ? 1 : kDim / 32;
#pragma unroll 1
    for (int piece = 0; piece < kDim / 32; piece += kPieces) {
      const auto column = [&](int i) {
        return 64 * ((piece + i) / 2) + 16 * t + 8 * ((piece + i) & 1);
      };
      uint32_t signs[kPieces] = {};  // bit e: column e reads an infinity; 8 + e: one below 0
#pragma unroll 1
      for (int key = first + g; key < end; key += 8) {
        const int row = static_cast<int>(fast_div(key, a.page_size));
        const int page = ld_int(table + row);
        if (!cache_page(page, a.pages)) continue;
        const int inside = key - row * static_cast<int>(a.page_size.divisor);
        const T* const src = head + page * a.v_page + inside * a.v_token;
        uint4 v[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          v[i] = column(i) < a.head_dim ? ld_ro(reinterpret_cast<const uint4*>(src + column(i)))
                                        : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t bits = word(v[i], e / 2) >> (16 * (e & 1)) & 0xffffu;
            const bool nan = (bits & 0x7fffu) > Mma<T>::kInfinity;  // as both infinities
            if (nan || bits == Mma<T>::kInfinity) signs[i] |= 1u << e;
            if (nan || bits == (0x8000u | Mma<T>::kInfinity)) signs[i] |= 0x100u << e;
          }
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) signs[i] |= __shfl_xor_sync(kFullMask, signs[i], x);
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          if (g + 8 * h >= unit.rows || !(l[h] > 0.0f)) continue;
#pragma unroll 1
          for (uint32_t left = (signs[i] | signs[i] >> 8) & 0xffu; left != 0; left &= left - 1) {
            const int e = __ffs(left) - 1;
            const uint32_t sign = signs[i] >> e & 0x101u;
            store(g + 8 * h, column(i) + e, sign == 1 ? INFINITY : sign == 0x100 ? -INFINITY : NAN);
          }
        }
      }
    }
  }

  // Calls write(row, column, eight values) for what the lane holds: rows g +
  // 8h; of piece c columns 8 (2t + x) + e in o[8c + e][2h + x].
  template <typename Write>
  __device__ __forceinline__ void each(const PagedArgs& a, const PagedUnit& unit, Write write) const {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int row = g + 8 * h;
      if (row >= unit.rows) continue;
#pragma unroll
      for (int c = 0; c < kDim / 64; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int d = 64 * c + 8 * (2 * t + x);
          if (d >= a.head_dim) continue;
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = o[8 * c + e][2 * h + x];
          write(h, row, d, y);
        }
    }
  }

  __device__ __forceinline__ void finish_whole(const PagedArgs& a, const PagedUnit& unit, int sequence,
                                               bool empty) {
    T* const dst = static_cast<T*>(a.out) +
                   (static_cast<int64_t>(sequence) * a.heads + unit.first_head) * a.head_dim;
    float f[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) f[h] = empty ? 0.0f : __fdividef(1.0f, l[h]);
    each(a, unit, [&](int h, int row, int d, const float (&y)[8]) {
      alignas(16) T z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) st_out(&z[e], y[e] * f[h]);
      *reinterpret_cast<uint4*>(dst + row * a.head_dim + d) = *reinterpret_cast<const uint4*>(z);
    });
  }

  __device__ __forceinline__ void finish_part(const PagedArgs& a, const PagedUnit& unit, float* part,
                                              int pitch, float* part_m, float* part_l) {
    each(a, unit, [&](int, int row, int d, const float (&y)[8]) {
      float4* const to = reinterpret_cast<float4*>(part + row * pitch + d);
      to[0] = make_float4(y[0], y[1], y[2], y[3]);
      to[1] = make_float4(y[4], y[5], y[6], y[7]);
    });
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      if (t == 0 && g + 8 * h < unit.rows) part_m[g + 8 * h] = m[h], part_l[g + 8 * h] = l[h];
  }
};

template <typename T, int kRows>
int pick_dim(const PagedArgs& a, cudaStream_t stream) {
  // Warps and stages by head size.  64: 12 x 2 at 168 registers (100,000 keys, 8
  // heads: 71 us; 8 x 3, 82 us; 16 x 2 the same as 12).  128: see
  // paged_stream.cuh.  Over 128 four warps of 32 to 36 KB of ring each, at 255
  // registers; 16 rows of 256 spill (184 bytes stored).
  if (a.head_dim <= 64) return paged_stream<MmaPolicy<T, 64, kRows>, 12, 2>(a, stream);
  if (a.head_dim <= 128) return paged_stream<MmaPolicy<T, 128, kRows>, 8, 2>(a, stream);
  if (a.head_dim <= 192) return paged_stream<MmaPolicy<T, 192, kRows>, 4, 3>(a, stream);
  return paged_stream<MmaPolicy<T, 256, kRows>, 4, 2>(a, stream);
}

}  // namespace

template <typename T>
int paged_attention_mma(const PagedArgs& a, cudaStream_t stream) {
  return a.group <= 8 ? pick_dim<T, 8>(a, stream) : pick_dim<T, 16>(a, stream);
}

template int paged_attention_mma<__half>(const PagedArgs&, cudaStream_t);
template int paged_attention_mma<__nv_bfloat16>(const PagedArgs&, cudaStream_t);

}  // namespace opl
