// What the kernels over a cache in pages share (pages.cu, paged_attn.cu): the cache as kernels get it, and the host's checks.
#pragma once
#include "ytc_common.cuh"

namespace ytk {

// Rows of new tokens [rows, heads, dim] in memory; strides in bytes.
struct PgRows {
  char* p;
  int64_t row, head;
};

// One pool of pages; strides in bytes.
struct PgPool {
  char* p;
  int64_t layer, page, head, row;
};

// Division of whole numbers below 2^31 by a divisor d the host knows: with 2^(l - 1) < d <= 2^l and m = floor(2^(31 + l) / d) + 1
// the error of n m / 2^(31 + l) is below 2^-l <= 1 / d, which the fraction of n / d leaves room for.
struct PgDiv {
  uint32_t mul, shift, d;
  __host__ __device__ __forceinline__ uint32_t of(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift); }
};
__host__ __device__ inline PgDiv pg_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return PgDiv{static_cast<uint32_t>((1ull << (31 + l)) / d + 1), 31 + l, d};
}

struct PgCache {
  PgPool k, v;
  PgDiv by_page, by_head;
  int32_t *table, *lens, *held, *refs, *status, *scratch;
  int layers, pages, page, heads, dim, slots, max_pages;
};

// Places in the scratch of a cache (int32 words).
struct PgScratch {
  int64_t ticket, copies, base, mark, src, dst, rows, held, lens, table, ids, number, words;
};
__host__ __device__ __forceinline__ PgScratch pg_scratch(int64_t slots, int64_t max_pages, int64_t pages) {
  PgScratch s;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t here = at;
    at += (n + 3) / 4 * 4;
    return here;
  };
  s.ticket = take(1);
  s.copies = take(1);
  s.base = take(slots + 1);
  s.mark = take(slots);
  s.src = take(slots);
  s.dst = take(slots);
  s.rows = take(slots);
  s.held = take(slots);
  s.lens = take(slots);
  s.table = take(slots * max_pages);
  s.ids = take(pages);
  s.number = take(pages);
  s.words = at;
  return s;
}

// Checks a cache that a caller hands in and turns its strides into bytes.
int pg_take(const char* who, const ytcuda_pages* c, PgCache* out);
// The rows of new tokens of a call, checked; `heads` of `dim` elements of `size` bytes.
int pg_rows(const char* who, const char* what, const void* p, const int64_t* strides, int size, PgRows* out);
// Elements of `size` bytes at p + sum of index * stride (in bytes): up to four axes, and `dim` elements in a row. And whether two of them have
// a byte in common.
struct PgBox {
  const char* p;
  int64_t extent[4], stride[4];
  int64_t dim;
};
bool pg_meet(const PgBox& a, const PgBox& b, int size);
inline PgBox pg_box(const PgPool& p, const PgCache& c) {
  return PgBox{p.p, {c.layers, c.pages, c.heads, c.page}, {p.layer, p.page, p.head, p.row}, c.dim};
}
// The widest of 16, 4 and 2 bytes in which rows of dim elements of these places can be copied.
inline int pg_width(uint64_t all_bits_or) { return all_bits_or % 16 == 0 ? 16 : all_bits_or % 4 == 0 ? 4 : 2; }
inline uint64_t pg_bits(const PgPool& p) {
  return reinterpret_cast<uint64_t>(p.p) | static_cast<uint64_t>(p.layer | p.page | p.head | p.row);
}
inline uint64_t pg_bits(const PgRows& r) { return reinterpret_cast<uint64_t>(r.p) | static_cast<uint64_t>(r.row | r.head); }

#ifdef __CUDACC__
// The page that holds position `at` of a slot; -1 where the slot holds none there.
__device__ __forceinline__ int pg_page_of(const PgCache& c, int slot, int64_t at) {
  if (at < 0 || at > 0x7fffffff) return -1;
  const int i = static_cast<int>(c.by_page.of(static_cast<uint32_t>(at)));
  if (i >= c.held[slot] || i >= c.max_pages) return -1;
  const int pg = c.table[static_cast<int64_t>(slot) * c.max_pages + i];
  return pg >= 0 && pg < c.pages ? pg : -1;
}
// Row of its page that position `at` has (at: not negative, below 2^31).
__device__ __forceinline__ int pg_row_of(const PgCache& c, int64_t at) {
  const uint32_t n = static_cast<uint32_t>(at);
  return static_cast<int>(n - c.by_page.of(n) * c.by_page.d);
}
// Every kernel here is launched so that it may be set up while the one in front of it in the stream still runs (about 1 us a launch),
// and begins with pg_begin(), before it reads or writes any memory. Only behind its own wait does a kernel let the next one in: what
// is behind that one in turn may rely on everything in front of this one being over.
__device__ __forceinline__ void pg_begin() {
  dependent_wait();
  dependent_trigger();
}
template <typename... KArgs, typename... Args>
cudaError_t pg_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  const bool was = overlap_scope();
  overlap_scope() = true;
  const cudaError_t e = launch_overlapped(kernel, grid, block, smem, st, static_cast<Args&&>(args)...);
  overlap_scope() = was;
  return e;
}
#endif

}  // namespace ytk
