// Paged decode attention on FP32 caches with rows on 16-byte boundaries (see
// paged_attention.cu for the operator), on FP32 units: no TF32.
//
// Bound by HBM for few query heads a key-value head (one operation a byte and
// head), by the FP32 units and shared memory from about eight on.  The tiles
// come through paged_stream.cuh, 16 keys at a time for heads of 64, else 8.
//
// * S = Q K^T: 2 or 4 lanes share a key, a part of its columns each, so that a
//   score takes one or two shuffles; they walk their 16-byte pieces in orders
//   that differ in the bits the swizzle leaves, free of bank conflicts.  Q is in
//   shared memory (read as broadcasts).  Packed fma.rn.f32x2.
// * O = P V: the lanes share the columns, and a weight is read, twice in a word
//   pair as the packed FMA wants it, by all lanes at once.
#include "paged_stream.cuh"

namespace opl {

namespace {

__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t x, uint64_t y) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(y));
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
struct Pairs {
  uint64_t x, y;
};
__device__ __forceinline__ Pairs ld_pairs(uint32_t src) {
  Pairs r;
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(r.x), "=l"(r.y) : "r"(src) : "memory");
  return r;
}
__device__ __forceinline__ uint64_t ld_pair(uint32_t src) {
  uint64_t r;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(r) : "r"(src) : "memory");
  return r;
}

// kDim: 64, 128 or 256.  kRows: the most query heads a unit.
template <int kDim_, int kRows_>
struct FmaPolicy {
  using T = float;
  static constexpr int kDim = kDim_, kRows = kRows_, kTile = kDim == 64 ? 16 : 8;
  static constexpr int kSplit = 32 / kTile;             // lanes of a key
  static constexpr int kPieceBytes = kTile * 128;       // 32 columns of all keys
  static constexpr int kLanePieces = kDim / 32 / kSplit;
  static constexpr int kPairs = kDim / 64;              // column pairs of a lane
  static constexpr bool kInfiniteValues = false;        // FP32 weights need no second look
  static constexpr int kQueryBytes = kRows * kDim * 4;
  static constexpr int kWarpShared = kQueryBytes + kRows * kTile * 8;  // and the weights

  float q_next[kRows][kDim / 32];
  uint64_t o[kRows][kPairs];
  float m[kRows], l[kRows];  // the same in all lanes; over this lane's key only
  int lane, key, sub;
  uint32_t query, weights;  // shared addresses
  float* shared;

  // The lane's columns: pairs 2 * lane, or 4 * lane (+ 128) and the next.
  __device__ __forceinline__ int column(int pair) const {
    return kPairs == 1 ? 2 * lane : 4 * lane + 2 * (pair & 1) + 128 * (pair >> 1);
  }

  __device__ __forceinline__ void init(int lane_, float* shared_) {
    lane = lane_, key = lane / kSplit, sub = lane % kSplit;
    shared = shared_;
    query = tc::smem_u32(shared);
    weights = query + kQueryBytes;
  }

  __device__ __forceinline__ void fetch_query(const PagedArgs& a, int sequence, int index) {
    const PagedUnit u = paged_unit<kRows>(a, index);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float* src =
          static_cast<const float*>(a.q) + sequence * a.q_batch + (u.first_head + r) * a.q_head;
#pragma unroll
      for (int i = 0; i < kDim / 32; ++i) {
        const int d = 32 * i + lane;
        q_next[r][i] = r < u.rows && d < a.head_dim ? ld_ro(src + d) : 0.0f;
      }
    }
  }

  __device__ __forceinline__ void start(const PagedArgs&, int, int) {
    __syncwarp();  // the last segment's queries have been read
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kDim / 32; ++i) shared[r * kDim + 32 * i + lane] = q_next[r][i];
#pragma unroll
      for (int p = 0; p < kPairs; ++p) o[r][p] = 0;
      m[r] = -INFINITY, l[r] = 0.0f;
    }
    __syncwarp();
  }

  template <bool kAllSeen>
  __device__ __forceinline__ void add_values(uint32_t values, uint32_t seen) {
    // Rolled when keys are missing: the last tile of a sequence.
#pragma unroll(kAllSeen ? kTile / 2 : 1)
    for (int j = 0; j < kTile; j += 2) {
      uint64_t v[2][kPairs];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!kAllSeen && (seen >> (j + i) & 1u) == 0) {  // what lies behind the length is no value
#pragma unroll
          for (int p = 0; p < kPairs; ++p) v[i][p] = 0;
          continue;
        }
        const uint32_t row = values + (j + i) * 128;
        const int swizzle = (j + i) & 7;
        if constexpr (kPairs == 1) {
          v[i][0] = ld_pair(row + (lane / 16) * kPieceBytes + ((lane % 16 / 2) ^ swizzle) * 16 +
                            (lane & 1) * 8);
        } else {
#pragma unroll
          for (int p = 0; p < kPairs; p += 2) {
            const Pairs two = ld_pairs(row + (lane / 8 + 2 * p) * kPieceBytes +
                                       ((lane % 8) ^ swizzle) * 16);
            v[i][p] = two.x, v[i][p + 1] = two.y;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const Pairs w = ld_pairs(weights + (r * kTile + j) * 8);
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
          fma2(o[r][p], w.x, v[0][p]);
          fma2(o[r][p], w.y, v[1][p]);
        }
      }
    }
  }

  __device__ __forceinline__ void step(const PagedArgs& a, uint32_t keys, uint32_t values,
                                       uint32_t seen) {
    uint64_t dot[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) dot[r] = 0;
#pragma unroll
    for (int p = 0; p < kLanePieces; ++p) {
      const int piece = sub * kLanePieces + p;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int chunk = c ^ (sub * (8 / kSplit));
        const Pairs k = ld_pairs(keys + piece * kPieceBytes + key * 128 + (chunk ^ (key & 7)) * 16);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const Pairs x = ld_pairs(query + r * kDim * 4 + piece * 128 + chunk * 16);
          fma2(dot[r], k.x, x.x);
          fma2(dot[r], k.y, x.y);
        }
      }
    }
    const bool there = (seen >> key & 1u) != 0;
    float s[kRows], top[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float2 two = unpack2(dot[r]);
      float x = two.x + two.y;
#pragma unroll
      for (int b = 1; b < kSplit; b <<= 1) x += __shfl_xor_sync(kFullMask, x, b);
      s[r] = there ? x * a.scale_log2 : -INFINITY;
      top[r] = s[r];
    }
#pragma unroll
    for (int b = kSplit; b < 32; b <<= 1)
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        top[r] = fmaxf(top[r], __shfl_xor_sync(kFullMask, top[r], b));
    __syncwarp();  // the last tile's weights have been read
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float m_new = fmaxf(m[r], top[r]);
      const float base = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: all weights 0
      if (m_new != m[r]) {  // in all lanes or in none
        const float alpha = paged_exp2(m[r] - base);
        const uint64_t alpha2 = pack2(alpha, alpha);
        l[r] *= alpha;
#pragma unroll
        for (int p = 0; p < kPairs; ++p) o[r][p] = mul2(o[r][p], alpha2);
        m[r] = m_new;
      }
      const float w = paged_exp2(s[r] - base);
      l[r] += w;
      if (sub == 0)
        *reinterpret_cast<float2*>(shared + kQueryBytes / 4 + (r * kTile + key) * 2) =
            make_float2(w, w);
    }
    __syncwarp();
    constexpr uint32_t kAll = (1u << kTile) - 1;
    if (seen == kAll)
      add_values<true>(values, seen);
    else
      add_values<false>(values, seen);
  }

  // Sums over the lanes of different keys.  True when no key has a weight, or a
  // score is no number.
  __device__ __forceinline__ bool settle() {
    bool none = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int b = kSplit; b < 32; b <<= 1) l[r] += __shfl_xor_sync(kFullMask, l[r], b);
      none |= !(l[r] > 0.0f);  // in all lanes
    }
    return none;
  }

  __device__ __forceinline__ void finish_whole(const PagedArgs& a, const PagedUnit& unit, int sequence,
                                               bool empty) {
    float* const dst = static_cast<float*>(a.out) +
                       (static_cast<int64_t>(sequence) * a.heads + unit.first_head) * a.head_dim;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= unit.rows) continue;
      const float f = empty ? 0.0f : 1.0f / l[r];
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const float2 y = unpack2(o[r][p]);
        if (column(p) < a.head_dim)
          *reinterpret_cast<float2*>(dst + r * a.head_dim + column(p)) = make_float2(y.x * f, y.y * f);
      }
    }
  }

  __device__ __forceinline__ void finish_part(const PagedArgs& a, const PagedUnit& unit, float* part,
                                              int pitch, float* part_m, float* part_l) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= unit.rows) continue;
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const float2 y = unpack2(o[r][p]);
        if (column(p) < a.head_dim)
          *reinterpret_cast<float2*>(part + r * pitch + column(p)) = y;
      }
      if (lane == 0) part_m[r] = m[r], part_l[r] = l[r];
    }
  }
};

// Eight rows, heads of up to 128 (11 sequences of 7098 keys, 64/4 heads of 128:
// 123 us against 170 us for FmaPolicy; 97 are the reading of keys and values for
// each of the two units of a head).  Reading Q for every key would keep shared
// memory busy three times as long as the products take, so the 8 lanes of a key group share its keys' columns and
// each takes 2 (heads of 64: 4) keys against one piece of Q; the transposing sum
// over them leaves row r's scores in lane r of the group, where its maximum, sum
// and exponentials are, one row a lane.
template <int kDim_>
struct FmaRowsPolicy {
  using T = float;
  static constexpr int kDim = kDim_, kRows = 8, kTile = kDim == 64 ? 16 : 8;
  static constexpr int kKeys = kTile / 4;               // of a lane, and of its group
  static constexpr int kPieceBytes = kTile * 128;       // 32 columns of all keys
  static constexpr int kChunks = kDim / 32;             // 16-byte pieces of a lane
  static constexpr int kPairs = kDim / 64;              // column pairs of a lane
  static constexpr bool kInfiniteValues = false;        // FP32 weights need no second look
  static constexpr int kQueryBytes = kRows * kDim * 4;
  static constexpr int kWarpShared = kQueryBytes + kRows * kTile * 4;  // and the weights

  float q_next[kRows][kDim / 32];
  uint64_t o[kRows][kPairs];
  float m, l;  // of row `sub`; l over this lane's keys only
  int lane, group, sub;
  uint32_t query, weights;  // shared addresses
  float* shared;

  __device__ __forceinline__ int column(int pair) const {
    return kPairs == 1 ? 2 * lane : 4 * lane + 2 * (pair & 1);
  }

  __device__ __forceinline__ void init(int lane_, float* shared_) {
    lane = lane_, group = lane >> 3, sub = lane & 7;
    shared = shared_;
    query = tc::smem_u32(shared);
    weights = query + kQueryBytes;
  }

  __device__ __forceinline__ void fetch_query(const PagedArgs& a, int sequence, int index) {
    const PagedUnit u = paged_unit<kRows>(a, index);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float* src =
          static_cast<const float*>(a.q) + sequence * a.q_batch + (u.first_head + r) * a.q_head;
#pragma unroll
      for (int i = 0; i < kDim / 32; ++i) {
        const int d = 32 * i + lane;
        q_next[r][i] = r < u.rows && d < a.head_dim ? ld_ro(src + d) : 0.0f;
      }
    }
  }

  __device__ __forceinline__ void start(const PagedArgs&, int, int) {
    __syncwarp();  // the last segment's queries have been read
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int i = 0; i < kDim / 32; ++i) shared[r * kDim + 32 * i + lane] = q_next[r][i];
#pragma unroll
      for (int p = 0; p < kPairs; ++p) o[r][p] = 0;
    }
    m = -INFINITY, l = 0.0f;
    __syncwarp();
  }

  template <bool kAllSeen>
  __device__ __forceinline__ void add_values(uint32_t values, uint32_t seen) {
    // Rolled when keys are missing: the last tile of a sequence.
#pragma unroll(kAllSeen ? kTile / 4 : 1)
    for (int j = 0; j < kTile; j += 4) {
      uint64_t v[4][kPairs];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!kAllSeen && (seen >> (j + i) & 1u) == 0) {  // what lies behind the length is no value
#pragma unroll
          for (int p = 0; p < kPairs; ++p) v[i][p] = 0;
          continue;
        }
        const uint32_t row = values + (j + i) * 128;
        const int swizzle = (j + i) & 7;
        if constexpr (kPairs == 1) {
          v[i][0] = ld_pair(row + (lane / 16) * kPieceBytes + ((lane % 16 / 2) ^ swizzle) * 16 +
                            (lane & 1) * 8);
        } else {
          const Pairs two = ld_pairs(row + (lane / 8) * kPieceBytes + ((lane % 8) ^ swizzle) * 16);
          v[i][0] = two.x, v[i][1] = two.y;
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const Pairs w = ld_pairs(weights + (r * kTile + j) * 4);
        const float2 low = unpack2(w.x), high = unpack2(w.y);
        const uint64_t w4[4] = {pack2(low.x, low.x), pack2(low.y, low.y), pack2(high.x, high.x),
                                pack2(high.y, high.y)};
#pragma unroll
        for (int p = 0; p < kPairs; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) fma2(o[r][p], w4[i], v[i][p]);
      }
    }
  }

  __device__ __forceinline__ void step(const PagedArgs& a, uint32_t keys, uint32_t values,
                                       uint32_t seen) {
    uint64_t dot[kRows][kKeys];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int k = 0; k < kKeys; ++k) dot[r][k] = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      // The lanes of a group read different 16 bytes of 128: of heads of 128,
      // lane s has pieces 4 (s & 1) .. + 3 of 128 bytes number s / 2, of 64 two
      // pieces of number s / 4.
      const int piece = kDim == 64 ? sub >> 2 : sub >> 1;
      const int chunk = kDim == 64 ? 2 * (sub & 3) + (c ^ (sub >> 2))
                                   : 4 * (sub & 1) + ((c + (sub >> 1)) & 3);
      Pairs k[kKeys];
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        const int key = group * kKeys + x;
        k[x] = ld_pairs(keys + piece * kPieceBytes + key * 128 + (chunk ^ (key & 7)) * 16);
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const Pairs x = ld_pairs(query + r * kDim * 4 + piece * 128 + chunk * 16);
#pragma unroll
        for (int y = 0; y < kKeys; ++y) {
          fma2(dot[r][y], k[y].x, x.x);
          fma2(dot[r][y], k[y].y, x.y);
        }
      }
    }
    // Sums over the group: after halving the rows three times lane s has row s.
    float s[kRows][kKeys];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
        const float2 two = unpack2(dot[r][k]);
        s[r][k] = two.x + two.y;
      }
#pragma unroll
    for (int half = 4; half > 0; half >>= 1) {
      const bool upper = (sub & half) != 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (r >= half) continue;
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const float give = upper ? s[r][k] : s[r + half][k];
          const float keep = upper ? s[r + half][k] : s[r][k];
          s[r][k] = keep + __shfl_xor_sync(kFullMask, give, half);
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      s[0][k] = (seen >> (group * kKeys + k) & 1u) != 0 ? s[0][k] * a.scale_log2 : -INFINITY;
      top = fmaxf(top, s[0][k]);
    }
    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 8));
    top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 16));
    const float m_new = fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: all weights 0
    if (__any_sync(kFullMask, m_new != m)) {
      const float alpha = paged_exp2(m - base);
      l *= alpha;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float row_alpha = __shfl_sync(kFullMask, alpha, r);
#pragma unroll
        for (int p = 0; p < kPairs; ++p) o[r][p] = mul2(o[r][p], pack2(row_alpha, row_alpha));
      }
      m = m_new;
    }
    __syncwarp();  // the last tile's weights have been read
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      const float w = paged_exp2(s[0][k] - base);
      l += w;
      shared[kQueryBytes / 4 + sub * kTile + group * kKeys + k] = w;
    }
    __syncwarp();
    constexpr uint32_t kAll = (1u << kTile) - 1;
    if (seen == kAll)
      add_values<true>(values, seen);
    else
      add_values<false>(values, seen);
  }

  // Sums over the groups.  True when no key has a weight, or a
  // score is no number.
  __device__ __forceinline__ bool settle() {
    l += __shfl_xor_sync(kFullMask, l, 8);
    l += __shfl_xor_sync(kFullMask, l, 16);
    return __any_sync(kFullMask, !(l > 0.0f));
  }

  __device__ __forceinline__ void finish_whole(const PagedArgs& a, const PagedUnit& unit, int sequence,
                                               bool empty) {
    float* const dst = static_cast<float*>(a.out) +
                       (static_cast<int64_t>(sequence) * a.heads + unit.first_head) * a.head_dim;
    const float f = empty ? 0.0f : 1.0f / l;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float row_f = __shfl_sync(kFullMask, f, r);
      if (r >= unit.rows) continue;
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const float2 y = unpack2(o[r][p]);
        if (column(p) < a.head_dim)
          *reinterpret_cast<float2*>(dst + r * a.head_dim + column(p)) =
              make_float2(y.x * row_f, y.y * row_f);
      }
    }
  }

  __device__ __forceinline__ void finish_part(const PagedArgs& a, const PagedUnit& unit, float* part,
                                              int pitch, float* part_m, float* part_l) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= unit.rows) continue;
#pragma unroll
      for (int p = 0; p < kPairs; ++p)
        if (column(p) < a.head_dim)
          *reinterpret_cast<float2*>(part + r * pitch + column(p)) = unpack2(o[r][p]);
    }
    if (lane < unit.rows) part_m[lane] = m, part_l[lane] = l;
  }
};

template <int kDim, int kWarps, int kStages>
int pick_rows(const PagedArgs& a, cudaStream_t stream) {
  if (a.group == 1) return paged_stream<FmaPolicy<kDim, 1>, kWarps, kStages>(a, stream);
  if (a.group == 2) return paged_stream<FmaPolicy<kDim, 2>, kWarps, kStages>(a, stream);
  // A lane holds rows * kDim / 32 columns of the output: four rows at most of
  // heads of 256.
  if constexpr (kDim < 256) {
    if (a.group > 4) return paged_stream<FmaRowsPolicy<kDim>, kWarps, kStages>(a, stream);
  }
  return paged_stream<FmaPolicy<kDim, 4>, kWarps, kStages>(a, stream);
}

}  // namespace

int paged_attention_f32(const PagedArgs& a, cudaStream_t stream) {
  if (a.head_dim <= 64) return pick_rows<64, 8, 2>(a, stream);
  if (a.head_dim <= 128) return pick_rows<128, 8, 2>(a, stream);
  return pick_rows<256, 4, 2>(a, stream);
}

}  // namespace opl
