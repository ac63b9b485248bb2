// Index arithmetic of the paged key-value cache, shared by the kernels and
// compiled by a plain C++ compiler too, so that its guards can be tested
// without a GPU.  No address is formed from an index that these functions
// have not accepted.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define OPL_HD __host__ __device__ __forceinline__
#else
#define OPL_HD inline
#endif

namespace opl {

// Codes for the device's watchdog word (opl_read_and_clear_watchdog).
constexpr int kBadSlot = 0x6b01;    // slot past the cache's last token
constexpr int kBadPage = 0x6b02;    // block-table entry outside the cache
constexpr int kBadLength = 0x6b03;  // negative length, or past the table's row

// Unsigned division by a divisor fixed at launch (Granlund and Montgomery,
// "Division by invariant integers using multiplication", PLDI 1994), exact
// for dividends below 2^31.
struct FastDiv {
  uint32_t divisor, multiplier, shift;
};

inline FastDiv make_fast_div(uint32_t divisor) {
  FastDiv f{divisor, 0, 0};
  while ((uint64_t{1} << f.shift) < divisor) ++f.shift;
  f.multiplier = static_cast<uint32_t>(
      ((uint64_t{1} << 32) * ((uint64_t{1} << f.shift) - divisor)) / divisor + 1);
  return f;
}

OPL_HD uint32_t fast_div(uint32_t n, const FastDiv& f) {
#ifdef __CUDA_ARCH__
  const uint32_t high = __umulhi(n, f.multiplier);
#else
  const uint32_t high = static_cast<uint32_t>((uint64_t{n} * f.multiplier) >> 32);
#endif
  return (high + n) >> f.shift;
}

// A token's place in the cache.  Returns 0 when `slot` names a token of the
// cache, -1 for a negative slot (a token that is not to be kept), else
// kBadSlot.
OPL_HD int cache_slot(int64_t slot, int64_t pages, int page_size, int64_t* page, int* inside) {
  if (slot < 0) return -1;
  const int64_t p = slot / page_size;
  if (p >= pages) return kBadSlot;
  *page = p;
  *inside = static_cast<int>(slot - p * page_size);
  return 0;
}

// Whether a block-table entry names a page of the cache.
OPL_HD bool cache_page(int entry, int64_t pages) { return entry >= 0 && entry < pages; }

// The keys of a sequence that can be read: its length, cut to [0, capacity of
// its block-table row].
OPL_HD int readable_length(int length, int max_pages, int page_size) {
  const int64_t capacity = static_cast<int64_t>(max_pages) * page_size;
  if (length < 0) return 0;
  return length < capacity ? length : static_cast<int>(capacity);
}

}  // namespace opl
