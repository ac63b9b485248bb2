// Rotary position embedding, alone (opl_rope_*) and on the way into a paged
// key-value cache (opl_kv_append_*).
//
// The first rot_dim elements of a head form rot_dim / 2 pairs, (i, i +
// rot_dim / 2) or (2i, 2i + 1); pair i of token t is turned by the angle
// positions[axis(i)][t] * inv_freq[i]:
//   (a, b) -> (a cos - b sin, a sin + b cos),
// with the sine negated for the inverse, which is the transposed matrix and
// so the gradient.  The remaining elements are copied.
//
// Angle: the product is formed in FP64, in turns, and its whole turns are
// removed before anything is rounded to FP32 -- at position 10^6 an FP32
// product is off by up to 0.03 radians.  The fraction, rounded once to FP32
// (relative 2^-24), goes through sincospif.
//
// Bound by HBM: every element is read and written once.  One warp owns a
// token, or for few tokens a range of its elements (a decode step of one
// token would otherwise walk all its heads with 32 lanes): the angles are
// computed once per warp, two pairs a lane at a head of 128, and shared by
// all heads through shared memory; the first loads are issued ahead of them.
#include <cuda_bf16.h>

#include "opl_common.cuh"
#include "paged_index.h"

namespace opl {

namespace {

constexpr int kWarps = 2;
constexpr int kMaxHeadDim = 256;
constexpr int kMaxPairs = kMaxHeadDim / 2;
constexpr int kMaxAxes = 4;
// Items (one or two vectors each) that a lane loads before it rotates any, and
// warps of an SM, which take 64 registers a thread for it.  32768 tokens of 32
// heads of 128, BF16: 86.0 us (0.95 of the HBM copy rate); with 4 items and 20
// warps 87.4, with 1 and 32 warps 92.8.
constexpr int kBatch = 2, kResidentWarps = 32;

template <typename T>
struct RopeArgs {
  const T *q, *k, *v;
  T *q_out, *k_cache, *v_cache;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
  int64_t kc_page, kc_token, kc_head, vc_page, vc_token, vc_head;
  const int64_t* slots;  // nullptr: no cache (opl_rope_*)
  int64_t pages;
  int page_size;
  const int64_t* positions;
  const float* inv_freq;
  int section_end[kMaxAxes];
  float sine_sign;
  int tokens, rot_dim, pair_items;
  int q_items, k_items, all_items;  // running ends of the token's items
  FastDiv row_items, v_row_items;
  int splits, split_items;  // warps per token, items of each
  int* watchdog;
};

template <int kBytes>
struct Words {
  uint32_t w[kBytes / 4];
};
template <>
struct Words<2> {
  unsigned short w[1];
};

// Coherent loads, kept after griddepcontrol.wait by volatile: the output may
// be the input.
__device__ __forceinline__ Words<16> ld_words(const void* p, Words<16>*) {
  Words<16> r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
               : "l"(p)
               : "memory");
  return r;
}
__device__ __forceinline__ Words<8> ld_words(const void* p, Words<8>*) {
  Words<8> r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(r.w[0]), "=r"(r.w[1])
               : "l"(p)
               : "memory");
  return r;
}
__device__ __forceinline__ Words<4> ld_words(const void* p, Words<4>*) {
  Words<4> r;
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p) : "memory");
  return r;
}
__device__ __forceinline__ Words<2> ld_words(const void* p, Words<2>*) {
  Words<2> r;
  asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];" : "=h"(r.w[0]) : "l"(p) : "memory");
  return r;
}
__device__ __forceinline__ void st_words(void* p, const Words<16>& r) {
  *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}
__device__ __forceinline__ void st_words(void* p, const Words<8>& r) {
  *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
}
__device__ __forceinline__ void st_words(void* p, const Words<4>& r) {
  *reinterpret_cast<uint32_t*>(p) = r.w[0];
}
__device__ __forceinline__ void st_words(void* p, const Words<2>& r) {
  *reinterpret_cast<unsigned short*>(p) = r.w[0];
}

__device__ __forceinline__ int64_t ld_index(const int64_t* p) {
  long long r;
  asm volatile("ld.global.s64 %0, [%1];" : "=l"(r) : "l"(p));
  return r;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float x, float* y) { *y = x; }
__device__ __forceinline__ void from_f32(float x, __half* y) { *y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }

template <typename T, int V>
union Pack {
  Words<V * static_cast<int>(sizeof(T))> words;
  T e[V];
  __device__ Pack() {}
};

// kAdjacent: an item is 2V consecutive elements holding V pairs; otherwise V
// elements of the first half and the V elements that pair with them.
template <typename T, int V, bool kAdjacent>
__global__ void __launch_bounds__(32 * kWarps, kResidentWarps / kWarps)
    rope_kernel(const RopeArgs<T> a) {
  // cos and sin of pair i at [i % V][i / V]: lanes with neighbouring items
  // read neighbouring words.
  __shared__ float2 turns[kWarps][kMaxPairs];
  using Vec = Pack<T, V>;
  constexpr int kVecBytes = V * static_cast<int>(sizeof(T));
  pdl_begin();

  const int lane = threadIdx.x & 31;
  float2* turn = turns[threadIdx.x >> 5];
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t token = warp / a.splits;
  if (token >= a.tokens) return;
  const int first = static_cast<int>(warp - token * a.splits) * a.split_items;
  const int last = min(first + a.split_items, a.all_items);
  if (first >= last) return;

  T *k_row = nullptr, *v_row = nullptr;  // the token's place in the cache
  if (a.slots != nullptr) {
    int64_t page;
    int inside;
    const int bad = cache_slot(ld_index(a.slots + token), a.pages, a.page_size, &page, &inside);
    if (bad == 0) {
      k_row = a.k_cache + page * a.kc_page + inside * a.kc_token;
      v_row = a.v_cache + page * a.vc_page + inside * a.vc_token;
    } else if (bad > 0 && lane == 0) {
      watchdog_trip(a.watchdog, bad);
    }
  }

  bool have_turns = false;
  int held = -1;  // the pair item whose cos and sin are in `cs`
  float2 cs[V];
  for (int base = first; base < last; base += 32 * kBatch) {
    Vec x[kBatch][2];
    T* dst[kBatch];
    int pair[kBatch];    // pair item, or -1: a plain copy of one vector
    int second[kBatch];  // offset of the item's second vector
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int item = base + 32 * u + lane;
      dst[u] = nullptr;
      pair[u] = -1;
      second[u] = 0;
      if (item >= last) continue;
      const T* src;
      int c;
      if (item < a.k_items) {
        const bool is_q = item < a.q_items;
        const int local = is_q ? item : item - a.q_items;
        const int head = static_cast<int>(fast_div(local, a.row_items));
        c = local - head * static_cast<int>(a.row_items.divisor);
        if (is_q) {
          src = a.q + token * a.q_token + head * a.q_head;
          dst[u] = a.q_out + token * a.out_token + head * a.out_head;
        } else {
          src = a.k + token * a.k_token + head * a.k_head;
          dst[u] = k_row == nullptr ? nullptr : k_row + head * a.kc_head;
        }
        int offset;
        if (c < a.pair_items) {
          pair[u] = c;
          offset = kAdjacent ? 2 * V * c : V * c;
          second[u] = kAdjacent ? V : a.rot_dim / 2;
        } else {
          offset = a.rot_dim + (c - a.pair_items) * V;
        }
        src += offset;
        if (dst[u] != nullptr) dst[u] += offset;
      } else {
        const int local = item - a.k_items;
        const int head = static_cast<int>(fast_div(local, a.v_row_items));
        c = local - head * static_cast<int>(a.v_row_items.divisor);
        src = a.v + token * a.v_token + head * a.v_head + c * V;
        dst[u] = v_row == nullptr ? nullptr : v_row + head * a.vc_head + c * V;
      }
      if (dst[u] == nullptr) continue;
      x[u][0].words = ld_words(src, static_cast<Words<kVecBytes>*>(nullptr));
      if (pair[u] >= 0)
        x[u][1].words = ld_words(src + second[u], static_cast<Words<kVecBytes>*>(nullptr));
    }
    if (!have_turns) {
      have_turns = true;
      for (int i = lane; i < a.rot_dim / 2; i += 32) {
        int axis = 0;
#pragma unroll
        for (int s = 0; s < kMaxAxes - 1; ++s) axis += i >= a.section_end[s];
        const double position =
            static_cast<double>(ld_index(a.positions + static_cast<int64_t>(axis) * a.tokens + token));
        constexpr double kTurnsPerRadian = 0.15915494309189533577;  // 1 / (2 pi)
        double t = position * static_cast<double>(ld_ro(a.inv_freq + i)) * kTurnsPerRadian;
        t -= rint(t);
        float s, c;
        sincospif(2.0f * static_cast<float>(t), &s, &c);
        turn[(i % V) * a.pair_items + i / V] = make_float2(c, a.sine_sign * s);
      }
      __syncwarp();
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (dst[u] == nullptr) continue;
      if (pair[u] >= 0) {
        if (pair[u] != held) {
          held = pair[u];
#pragma unroll
          for (int e = 0; e < V; ++e) cs[e] = turn[e * a.pair_items + held];
        }
        Vec y[2];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int i0 = kAdjacent ? (2 * e) / V : 0, e0 = kAdjacent ? (2 * e) % V : e;
          const int i1 = kAdjacent ? (2 * e + 1) / V : 1, e1 = kAdjacent ? (2 * e + 1) % V : e;
          const float p = to_f32(x[u][i0].e[e0]), r = to_f32(x[u][i1].e[e1]);
          from_f32(p * cs[e].x - r * cs[e].y, &y[i0].e[e0]);
          from_f32(p * cs[e].y + r * cs[e].x, &y[i1].e[e1]);
        }
        st_words(dst[u], y[0].words);
        st_words(dst[u] + second[u], y[1].words);
      } else {
        st_words(dst[u], x[u][0].words);
      }
    }
  }
}

bool fits(int vector, const void* p, std::initializer_list<int64_t> strides, size_t size) {
  if (reinterpret_cast<std::uintptr_t>(p) % (vector * size) != 0) return false;
  for (int64_t s : strides)
    if (s % vector != 0) return false;
  return true;
}

// Fills what follows from the shape and launches.  The widest vector (16, 8
// or sizeof(T) bytes) that divides every address, stride and section of a
// head is taken.
template <typename T>
int launch_rope(RopeArgs<T> a, int heads, int kv_heads, int head_dim, const opl_rope_spec* rope,
                cudaStream_t stream) {
  a.rot_dim = rope->rot_dim;
  a.positions = rope->positions;
  a.inv_freq = rope->inv_freq;
  a.sine_sign = rope->inverse != 0 ? -1.0f : 1.0f;
  int end = 0;
  for (int s = 0; s < kMaxAxes; ++s) {
    end += s < rope->axes ? rope->sections[s] : 0;
    a.section_end[s] = end;
  }
  const auto usable = [&](int vector) {
    const size_t size = sizeof(T);
    return head_dim % vector == 0 && a.rot_dim % (2 * vector) == 0 &&
           fits(vector, a.q, {a.q_token, a.q_head}, size) &&
           fits(vector, a.q_out, {a.out_token, a.out_head}, size) &&
           fits(vector, a.k, {a.k_token, a.k_head}, size) &&
           fits(vector, a.v, {a.v_token, a.v_head}, size) &&
           fits(vector, a.k_cache, {a.kc_page, a.kc_token, a.kc_head}, size) &&
           fits(vector, a.v_cache, {a.vc_page, a.vc_token, a.vc_head}, size);
  };
  const int wide = 16 / static_cast<int>(sizeof(T));
  const int vector = usable(wide) ? wide : usable(wide / 2) ? wide / 2 : 1;
  a.pair_items = a.rot_dim / 2 / vector;
  const int row_items = a.pair_items + (head_dim - a.rot_dim) / vector;
  const int v_row_items = head_dim / vector;
  const int64_t items = (int64_t{heads} + kv_heads) * row_items + int64_t{kv_heads} * v_row_items;
  if (items > (int64_t{1} << 30)) return cudaErrorInvalidValue;
  if (a.slots != nullptr) {
    a.watchdog = watchdog_word();
    if (a.watchdog == nullptr) return cudaErrorInvalidDevice;
  }
  a.row_items = make_fast_div(row_items);
  a.v_row_items = make_fast_div(v_row_items);
  a.q_items = heads * row_items;
  a.k_items = a.q_items + kv_heads * row_items;
  a.all_items = static_cast<int>(items);
  // Few tokens: split a token's items over warps, as many as are resident at
  // once or one more, whichever takes fewer batches one after the other (1023
  // tokens of 36 FP32 heads of 80: 7.7 us with 4 warps a token, 8.7 with 5, a
  // second wave; 4097 of 12 of 64: 6.5 us with 2, 7.3 with 1).
  const int rounds = (a.all_items + 31) / 32;
  const int64_t resident = static_cast<int64_t>(sm_count()) * kResidentWarps;
  const auto per_warp = [&](int64_t splits) {
    return splits >= rounds ? 1 : static_cast<int>((rounds + splits - 1) / splits);
  };
  const auto batches = [&](int64_t splits) {
    return (a.tokens * splits + resident - 1) / resident * ((per_warp(splits) + kBatch - 1) / kBatch);
  };
  int64_t splits = 1;
  if (a.tokens <= resident) {
    splits = resident / a.tokens;
    if (batches(splits + 1) <= batches(splits)) ++splits;
  }
  const int per = per_warp(splits);
  a.split_items = 32 * per;
  a.splits = (rounds + per - 1) / per;
  const int64_t blocks = (static_cast<int64_t>(a.tokens) * a.splits + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;

  const bool adjacent = rope->adjacent != 0;
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * kWarps);
  constexpr int kWide = 16 / static_cast<int>(sizeof(T));
  cudaError_t error;
  if (vector == kWide)
    error = adjacent ? launch_pdl(rope_kernel<T, kWide, true>, grid, block, stream, a)
                     : launch_pdl(rope_kernel<T, kWide, false>, grid, block, stream, a);
  else if (vector == kWide / 2)
    error = adjacent ? launch_pdl(rope_kernel<T, kWide / 2, true>, grid, block, stream, a)
                     : launch_pdl(rope_kernel<T, kWide / 2, false>, grid, block, stream, a);
  else
    error = adjacent ? launch_pdl(rope_kernel<T, 1, true>, grid, block, stream, a)
                     : launch_pdl(rope_kernel<T, 1, false>, grid, block, stream, a);
  return error != cudaSuccess ? error : cudaGetLastError();
}

bool valid_rope(const opl_rope_spec* rope, int head_dim) {
  if (rope == nullptr || rope->rot_dim < 0 || rope->rot_dim > head_dim || rope->rot_dim % 2 != 0)
    return false;
  if (rope->rot_dim == 0) return true;
  if (rope->positions == nullptr || rope->inv_freq == nullptr || rope->axes < 1 ||
      rope->axes > kMaxAxes)
    return false;
  int64_t pairs = 0;
  for (int s = 0; s < rope->axes; ++s) {
    if (rope->sections[s] < 0) return false;
    pairs += rope->sections[s];
  }
  return pairs == rope->rot_dim / 2;
}

template <typename T>
int rope(const void* x, void* out, int tokens, int heads, int head_dim, int64_t x_token,
         int64_t x_head, int64_t out_token, int64_t out_head, const opl_rope_spec* spec,
         cudaStream_t stream) {
  if (x == nullptr || out == nullptr || tokens <= 0 || heads <= 0 || head_dim <= 0 ||
      head_dim > kMaxHeadDim || !valid_rope(spec, head_dim))
    return cudaErrorInvalidValue;
  RopeArgs<T> a = {};
  a.q = static_cast<const T*>(x);
  a.q_out = static_cast<T*>(out);
  a.q_token = x_token;
  a.q_head = x_head;
  a.out_token = out_token;
  a.out_head = out_head;
  a.tokens = tokens;
  return launch_rope(a, heads, 0, head_dim, spec, stream);
}

template <typename T>
int kv_append(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
              int64_t k_head, const void* v, int64_t v_token, int64_t v_head, void* q_out,
              int64_t out_token, int64_t out_head, const opl_kv_cache* cache, const int64_t* slots,
              int tokens, int heads, const opl_rope_spec* spec, cudaStream_t stream) {
  if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || cache == nullptr ||
      cache->k == nullptr || cache->v == nullptr || cache->k == cache->v || slots == nullptr ||
      tokens <= 0 || heads <= 0 || cache->pages <= 0 || cache->page_size <= 0 ||
      cache->kv_heads <= 0 || cache->head_dim <= 0 || cache->head_dim > kMaxHeadDim ||
      !valid_rope(spec, cache->head_dim))
    return cudaErrorInvalidValue;
  RopeArgs<T> a = {};
  a.q = static_cast<const T*>(q);
  a.k = static_cast<const T*>(k);
  a.v = static_cast<const T*>(v);
  a.q_out = static_cast<T*>(q_out);
  a.k_cache = static_cast<T*>(cache->k);
  a.v_cache = static_cast<T*>(cache->v);
  a.q_token = q_token;
  a.q_head = q_head;
  a.k_token = k_token;
  a.k_head = k_head;
  a.v_token = v_token;
  a.v_head = v_head;
  a.out_token = out_token;
  a.out_head = out_head;
  a.kc_page = cache->k_page;
  a.kc_token = cache->k_token;
  a.kc_head = cache->k_head;
  a.vc_page = cache->v_page;
  a.vc_token = cache->v_token;
  a.vc_head = cache->v_head;
  a.slots = slots;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.tokens = tokens;
  return launch_rope(a, heads, cache->kv_heads, cache->head_dim, spec, stream);
}

}  // namespace

}  // namespace opl

#define OPL_ROPE_ENTRY(SUFFIX, ABI_T, T)                                                         \
  int opl_rope_##SUFFIX(const ABI_T* x, ABI_T* out, int tokens, int heads, int head_dim,         \
                        int64_t x_token, int64_t x_head, int64_t out_token, int64_t out_head,    \
                        const opl_rope_spec* rope, opl_stream_t stream) {                        \
    return opl::rope<T>(x, out, tokens, heads, head_dim, x_token, x_head, out_token, out_head,   \
                        rope, stream);                                                           \
  }                                                                                              \
  int opl_kv_append_##SUFFIX(const ABI_T* q, int64_t q_token, int64_t q_head, const ABI_T* k,    \
                             int64_t k_token, int64_t k_head, const ABI_T* v, int64_t v_token,   \
                             int64_t v_head, ABI_T* q_out, int64_t out_token, int64_t out_head,  \
                             const opl_kv_cache* cache, const int64_t* slots, int tokens,        \
                             int heads, const opl_rope_spec* rope, opl_stream_t stream) {        \
    return opl::kv_append<T>(q, q_token, q_head, k, k_token, k_head, v, v_token, v_head, q_out,  \
                             out_token, out_head, cache, slots, tokens, heads, rope, stream);    \
  }

extern "C" {
OPL_ROPE_ENTRY(f32, float, float)
OPL_ROPE_ENTRY(f16, opl_half_t, __half)
OPL_ROPE_ENTRY(bf16, opl_bf16_t, __nv_bfloat16)
}
