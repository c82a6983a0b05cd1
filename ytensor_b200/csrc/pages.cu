// A cache in pages: handing out pages, storing rows, forking, keeping accepted rows, compacting the pool.
//
// All of it is copying and counting. The counting (which pages are free, who holds one) is whole numbers of a few KB and runs
// in one CTA or one per slot, so that its results do not depend on any order; the copying runs on the whole GPU, a warp for a
// piece of at most 4 KB with eight 16-byte loads of a lane in flight before the first store. A call that counts and copies is
// two kernels, the second launched while the first one runs (programmatic dependent launch).
#include "pages.cuh"
#include "ptx_sm100.cuh"

namespace ytk {

constexpr int PG_WARPS = 8;      // warps per CTA of the copying kernels
constexpr int PG_UNROLL = 8;     // pieces of a row that a lane has in flight
constexpr int PG_COUNT = 1024;   // threads of the counting kernels

template <int BYTES>
struct PgWord;
template <>
struct PgWord<16> {
  using type = uint4;
};
template <>
struct PgWord<4> {
  using type = uint32_t;
};
template <>
struct PgWord<2> {
  using type = uint16_t;
};

__device__ __forceinline__ void pg_flag(const PgCache& c, int bit) { atomicOr(c.status, bit); }

// Sum of the values of the threads in front, and of all (PG_COUNT threads).
__device__ __forceinline__ int pg_scan(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (`sums` may still be read from the call before)
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int w = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return x - v + (warp ? before : 0);
}

// The warp copies `rows` rows of `words` words each.
template <typename W>
__device__ __forceinline__ void pg_copy_rows(char* dst, int64_t dst_row, const char* src, int64_t src_row, int rows, int words) {
  const int lane = threadIdx.x & 31;
  const int n = rows * words;
  const bool whole = dst_row == words * static_cast<int64_t>(sizeof(W)) && src_row == dst_row;
  for (int i0 = lane; i0 < n; i0 += 32 * PG_UNROLL) {
    W w[PG_UNROLL];
#pragma unroll
    for (int u = 0; u < PG_UNROLL; ++u) {
      const int i = i0 + 32 * u;
      if (i < n) {
        const int r = whole ? 0 : i / words;
        w[u] = *reinterpret_cast<const W*>(src + r * src_row + (i - r * words) * static_cast<int64_t>(sizeof(W)));
      }
    }
#pragma unroll
    for (int u = 0; u < PG_UNROLL; ++u) {
      const int i = i0 + 32 * u;
      if (i < n) {
        const int r = whole ? 0 : i / words;
        *reinterpret_cast<W*>(dst + r * dst_row + (i - r * words) * static_cast<int64_t>(sizeof(W))) = w[u];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- append
// A warp stores what `run` new rows hold of one head in keys or values: in the pages that is one stretch of up to 4 KB, and the warps
// beside it take the other heads of the same rows. A lane finds where each row goes (five reads that depend on one another), for
// the next item while this one's words are on their way. The row's slot: the last one that starts at or before it. Four prompts of up to
// 8000 rows, fp32, 309 MB in and out: 54 us, 5.7 TB/s (65 us with three CTAs an SM instead of four).
template <int BYTES>
__global__ void __launch_bounds__(PG_WARPS * 32, 4) pages_append_kernel(const PgCache c, const PgRows k, const PgRows v, const int32_t* starts,
                                                                     int rows, int layer, PgDiv by_words, int run) {
  using W = typename PgWord<BYTES>::type;
  pg_begin();
  const int lane = threadIdx.x & 31, warps = gridDim.x * PG_WARPS, row_words = by_words.d;
  const int first = max(0, starts[0]), last = min(rows, starts[c.slots]);
  const int items = (rows + run - 1) / run * 2 * c.heads;
  const auto part = [&](int item, int* row0, int* head) {  // and whether it is of values
    const int x = static_cast<int>(c.by_head.of(item));
    *head = item - x * c.heads;
    *row0 = (x >> 1) * run;
    return (x & 1) != 0;
  };
  const auto find = [&](int item) -> unsigned long long {
    int row0, head;
    if (item >= items) return 0;
    const PgPool& pool = part(item, &row0, &head) ? c.v : c.k;
    const int row = row0 + lane;
    if (lane >= run || row < first || row >= last) return 0;
    int lo = 0, hi = c.slots;  // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (starts[mid] <= row ? lo : hi) = mid;
    }
    const int64_t at = static_cast<int64_t>(c.lens[lo]) + (row - starts[lo]);
    const int pg = pg_page_of(c, lo, at);
    if (pg < 0 || c.refs[pg] != 1) {
      pg_flag(c, pg < 0 ? YTC_PAGES_INVALID : YTC_PAGES_SHARED);
      return 0;
    }
    return reinterpret_cast<unsigned long long>(pool.p + layer * pool.layer + pg * pool.page + head * pool.head + pg_row_of(c, at) * pool.row);
  };
  int item = blockIdx.x * PG_WARPS + (threadIdx.x >> 5);
  unsigned long long to = find(item);
  for (; item < items; item += warps) {
    int row0, head;
    const PgRows& src = part(item, &row0, &head) ? v : k;
    const char* const from = src.p + row0 * src.row + head * src.head;
    unsigned long long next = 0;
    for (int w0 = 0; w0 < run * row_words; w0 += 32 * PG_UNROLL) {  // (more than one round only where one row takes it)
      W w[PG_UNROLL];
      char* dst[PG_UNROLL];
#pragma unroll
      for (int u = 0; u < PG_UNROLL; ++u) {
        const int i = w0 + lane + 32 * u, r = static_cast<int>(by_words.of(i)), x = i - r * row_words;
        dst[u] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, to, r & 31));
        if (r >= run) dst[u] = nullptr;
        if (dst[u]) {
          w[u] = *reinterpret_cast<const W*>(from + r * src.row + x * static_cast<int64_t>(sizeof(W)));
          dst[u] += x * static_cast<int64_t>(sizeof(W));
        }
      }
      if (w0 == 0) next = find(item + warps);
#pragma unroll
      for (int u = 0; u < PG_UNROLL; ++u)
        if (dst[u]) *reinterpret_cast<W*>(dst[u]) = w[u];
    }
    to = next;
  }
}

// ---------------------------------------------------------------------------------------------- reserve
// One CTA: what each slot wants, the free pages in ascending order, and who gets which. A page that a slot holds already is replaced where
// new positions go to it and others hold it too: the one that position lens falls in, whose rows in front of lens are copied, and those
// behind it, which only a shortened sequence has. Seven reads that depend on one another, 6 us; refs are read once, 32 KB a round, until
// enough free pages are found.
__device__ __forceinline__ bool pg_shared(const PgCache& c, int slot, int i) {
  const int pg = c.table[static_cast<int64_t>(slot) * c.max_pages + i];
  return pg >= 0 && pg < c.pages && c.refs[pg] > 1;
}
// Who gets which where some slot has such pages behind the first: apart from the kernel, whose code is fetched while it runs (a fork and
// a reserve of four beams: 11.9 us, 12.2 with all of it in one loop). refs says who shares what until all slots are through: only
// then those of the replaced pages go down.
__device__ __noinline__ void pg_hand_out(const PgCache& c, const int32_t* counts, int* n_copies, int* n_left) {
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  int32_t* const left = c.scratch + at.number;  // pages that are replaced, one for each new one at most
  const int t = threadIdx.x, lane = t & 31;
  for (int s = t >> 5; s < c.slots; s += PG_COUNT / 32) {  // a warp a slot
    const int len = c.lens[s], held = c.held[s], count = counts[s];
    if (count <= 0 || c.scratch[at.mark + s] == -2) continue;
    const int first = static_cast<int>(c.by_page.of(len)), need = static_cast<int>(c.by_page.of(static_cast<uint32_t>(len) + count - 1)) + 1;
    int k = c.scratch[at.base + s];
#pragma unroll 1
    for (int i0 = first; i0 < need; i0 += 32) {
      const int i = i0 + lane;
      const bool replaced = i < min(need, held) && pg_shared(c, s, i), takes = replaced || (i >= held && i < need);
      const unsigned all = __ballot_sync(0xffffffffu, takes);
      if (takes) {
        int32_t* const entry = c.table + static_cast<int64_t>(s) * c.max_pages + i;
        const int old = *entry, id = c.scratch[at.ids + k + __popc(all & ((1u << lane) - 1))], rows = i == first ? pg_row_of(c, len) : 0;
        *entry = id;
        c.refs[id] = 1;
        if (replaced) left[atomicAdd(n_left, 1)] = old;
        if (replaced && rows) {
          const int n = atomicAdd(n_copies, 1);
          c.scratch[at.src + n] = old;
          c.scratch[at.dst + n] = id;
          c.scratch[at.rows + n] = rows;
        }
      }
      k += __popc(all);
    }
    __syncwarp();
    if (lane == 0 && need > held) c.held[s] = need;
  }
  __syncthreads();
  for (int i = t; i < *n_left; i += PG_COUNT) atomicSub(c.refs + left[i], 1);
}
// How many of the entries from .. to - 1 of this thread's slot others hold too, for sequences that are written anew: in pieces of 128, dealt to
// the warps (64 slots of 500 pages each 23 us, with a thread a slot 121).
__device__ __noinline__ int pg_count_shared(const PgCache& c, int s0, int from, int to, int (*behind)[PG_COUNT]) {
  const int t = threadIdx.x, lane = t & 31;
  behind[0][t] = from;
  behind[1][t] = to;
  behind[2][t] = 0;
  __syncthreads();
  for (int l = 0, turn = t >> 5; l < min(PG_COUNT, c.slots - s0); ++l) {
    const int begin = behind[0][l], end = behind[1][l], pieces = max(0, end - begin + 127) / 128;
    for (; turn < pieces; turn += PG_COUNT / 32) {
      int n = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = begin + 128 * turn + 32 * u + lane;
        if (i < end) n += pg_shared(c, s0 + l, i);
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (n && lane == 0) atomicAdd(&behind[2][l], n);
    }
    turn -= pieces;
  }
  __syncthreads();
  return behind[2][t];
}
__global__ void __launch_bounds__(PG_COUNT) pages_reserve_kernel(const __grid_constant__ PgCache c, const int32_t* counts) {
  pg_begin();
  __shared__ int sums[32];
  __shared__ int behind[3][PG_COUNT], many[2];  // many: some slot of a round has more such pages than a thread counts by itself
  __shared__ int bad, n_copies, n_left, deep;  // deep: some slot replaces more pages than its first one
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  int32_t* const base = c.scratch + at.base;
  int32_t* const mark = c.scratch + at.mark;
  int32_t* const ids = c.scratch + at.ids;
  const int t = threadIdx.x;
  if (t == 0) bad = n_copies = n_left = deep = many[0] = many[1] = 0;
  __syncthreads();
  int want_all = 0;
  for (int s0 = 0; s0 < c.slots; s0 += PG_COUNT) {
    const int s = s0 + t;
    int want = 0, from = 0, to = 0;  // from, to: entries behind the first that are held already and written now
    if (s < c.slots) {
      const int len = c.lens[s], held = c.held[s], count = counts[s];
      mark[s] = -1;
      if (count) {
        bool ok = count > 0 && len >= 0 && held >= 0 && held <= c.max_pages;
        const uint32_t end = static_cast<uint32_t>(ok ? len : 0) + static_cast<uint32_t>(ok ? count : 0) - 1;  // the last new position
        const int64_t need = !ok ? 0 : end > 0x7fffffffu ? (1ll << 31) : static_cast<int64_t>(c.by_page.of(end)) + 1;
        const int first = static_cast<int>(c.by_page.of(ok ? len : 0));
        int copy = -1;
        const int pg = ok ? pg_page_of(c, s, len) : -1;
        if (pg >= 0) copy = c.refs[pg] > 1 ? pg : -1;
        else ok = ok && !pg_row_of(c, len);
        ok = ok && first <= held;  // (the positions that are written have their pages)
        if (!ok) {
          pg_flag(c, YTC_PAGES_INVALID);
          mark[s] = -2;
        } else if (need > c.max_pages) {
          bad = 1;
        } else {
          mark[s] = copy;
          want = (need > held ? static_cast<int>(need) - held : 0) + (copy >= 0);
          from = first + 1;
          to = min(static_cast<int>(need), held);
#pragma unroll 1
          for (; from < to && to - from <= 4; ++from)
            if (pg_shared(c, s, from)) {
              ++want;
              deep = 1;
            }
        }
      }
    }
    if (from < to) many[s0 / PG_COUNT % 2] = 1;
    int total, before = pg_scan(want, sums, &total);
    if (many[s0 / PG_COUNT % 2]) {  // (behind the barriers of the sum; a round later the other one is set)
      const int more = pg_count_shared(c, s0, from, to, behind);
      if (more) deep = 1;
      before = pg_scan(want += more, sums, &total);
    }
    if (s < c.slots) base[s] = want_all + before;
    want_all += total;
  }
  if (t == 0) base[c.slots] = want_all;
  // the first want_all free pages
  int found = 0;
  const bool wide = reinterpret_cast<uintptr_t>(c.refs) % 16 == 0;
  for (int p0 = 0; p0 < c.pages && found < want_all; p0 += 8 * PG_COUNT) {
    const int p = p0 + 8 * t;
    int32_t r[8];
    if (wide && p + 8 <= c.pages) {
      *reinterpret_cast<int4*>(r) = *reinterpret_cast<const int4*>(c.refs + p);
      *reinterpret_cast<int4*>(r + 4) = *reinterpret_cast<const int4*>(c.refs + p + 4);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) r[u] = p + u < c.pages ? c.refs[p + u] : 1;
    }
    int n = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) n += r[u] == 0;
    int total;
    int k = found + pg_scan(n, sums, &total);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (r[u] == 0) {
        if (k < want_all) ids[k] = p + u;
        ++k;
      }
    found += total;
  }
  __syncthreads();
  const bool full = bad || found < want_all;
  if (full) {
    if (t == 0) {
      pg_flag(c, YTC_PAGES_FULL);
      c.scratch[at.copies] = 0;
    }
    return;
  }
  if (deep) {
    pg_hand_out(c, counts, &n_copies, &n_left);
    if (t == 0) c.scratch[at.copies] = n_copies;
    return;
  }
  for (int s = t >> 5; s < c.slots; s += PG_COUNT / 32) {  // a warp a slot
    const int from = base[s], want = base[s + 1] - from, old = mark[s], len = c.lens[s], held = c.held[s], count = counts[s];
    if (count <= 0 || old == -2) continue;
    const bool copy = old >= 0;
    for (int k = t & 31; k < want; k += 32) {
      const int id = ids[from + k], i = copy && k == 0 ? static_cast<int>(c.by_page.of(len)) : held + k - copy;
      c.table[static_cast<int64_t>(s) * c.max_pages + i] = id;
      c.refs[id] = 1;
      if (copy && k == 0) {
        const int n = atomicAdd(&n_copies, 1);
        c.scratch[at.src + n] = old;
        c.scratch[at.dst + n] = id;
        c.scratch[at.rows + n] = pg_row_of(c, len);  // (none where lens falls between pages)
        atomicSub(c.refs + old, 1);
      }
    }
    __syncwarp();
    if ((t & 31) == 0 && want > copy) c.held[s] = held + want - copy;
  }
  __syncthreads();
  if (t == 0) c.scratch[at.copies] = n_copies;
}

// A warp copies up to 4 KB of the rows of one head, layer and pool of a page. 64 beams of eight searches, 12 layers, 61 MB: 12 us.
template <int BYTES>
__global__ void __launch_bounds__(PG_WARPS * 32) pages_copy_kernel(const PgCache c, int row_words) {
  using W = typename PgWord<BYTES>::type;
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  pg_begin();
  const int rows_a_piece = max(1, 32 * PG_UNROLL / row_words), pieces = (c.page + rows_a_piece - 1) / rows_a_piece;
  const int64_t per_copy = 2ll * c.layers * c.heads * pieces;
  const int64_t items = c.scratch[at.copies] * per_copy, warps = static_cast<int64_t>(gridDim.x) * PG_WARPS;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * PG_WARPS + (threadIdx.x >> 5); item < items; item += warps) {
    const int n = static_cast<int>(item / per_copy);
    int rest = static_cast<int>(item - n * per_copy);
    const int first = rest % pieces * rows_a_piece, rows = min(rows_a_piece, c.scratch[at.rows + n] - first);
    if (rows <= 0) continue;
    rest /= pieces;
    const PgPool& pool = rest & 1 ? c.v : c.k;
    rest >>= 1;
    char* const p = pool.p + rest / c.heads * pool.layer + rest % c.heads * pool.head + first * pool.row;
    pg_copy_rows<W>(p + c.scratch[at.dst + n] * pool.page, pool.row, p + c.scratch[at.src + n] * pool.page, pool.row, rows, row_words);
  }
}

// ---------------------------------------------------------------------------------------------- keep
// Whether the accepted rows of a slot can move (the same answer in every lane of the warp).
__device__ __forceinline__ int pg_keep_bad(const PgCache& c, int s, int64_t base, int n, const int32_t* accepted, int depth) {
  const int lane = threadIdx.x & 31;
  int bad = n < 0 || base < 0 || (accepted && n > depth) ? YTC_PAGES_INVALID : 0;
  if (base + n > static_cast<int64_t>(c.held[s]) * c.page) bad = YTC_PAGES_INVALID;
  if (!bad && accepted)
    for (int j = lane; j < n; j += 32) {
      const int a = accepted[static_cast<int64_t>(s) * depth + j];
      const int b = j ? accepted[static_cast<int64_t>(s) * depth + j - 1] : -1;
      const int to = pg_page_of(c, s, base + j);
      if (a <= b || to < 0 || pg_page_of(c, s, base + a) < 0) bad |= YTC_PAGES_INVALID;
      else if (a != j && c.refs[to] != 1) bad |= YTC_PAGES_SHARED;
    }
  return __reduce_or_sync(0xffffffffu, bad);
}

// A CTA moves the accepted rows of one slot in some of its layers, heads and pools, a warp each: where the rows lie is worked out
// once for up to PG_MOVES of them. Rows only move down and in ascending order, so a batch that has been read before it is written
// never hides a row of a later batch. The CTA that finishes last writes the lengths: every other one has read them by then. 64 slots, up
// to 12 of 48 rows in 28 layers, 72 MB in rows of 256 bytes: 27 us. Bound by reads that depend on one another in front of the first row,
// not by memory: of 10 layers the SMs are active half of the time and DRAM is at 6 %.
constexpr int PG_MOVES = 128;
template <int BYTES>
__global__ void __launch_bounds__(PG_WARPS * 32, 3) pages_keep_kernel(const PgCache c, const int32_t* kept, const int32_t* accepted,
                                                                   int depth, const int32_t* base, PgDiv by_words) {
  using W = typename PgWord<BYTES>::type;
  __shared__ int page[2][PG_MOVES], row[2][PG_MOVES];  // from, to
  __shared__ PgDiv by_moves;
  __shared__ int last;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int items = 2 * c.layers * c.heads, s = blockIdx.x;
  pg_begin();
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  const int n = kept[s];
  const int64_t b = base ? base[s] : c.lens[s];
  const int bad = pg_keep_bad(c, s, b, n, accepted, depth);  // (the same in every warp)
  if (blockIdx.y == 0 && t == 0) c.scratch[at.mark + s] = bad;
  if (accepted && n > 0 && !bad) {
    const int32_t* const mine = accepted + static_cast<int64_t>(s) * depth;
    for (int j0 = 0; j0 < n; j0 += PG_MOVES) {
      const int moves = min(PG_MOVES, n - j0);
      __syncthreads();
      for (int i = t; i < 2 * moves; i += PG_WARPS * 32) {
        const int j = i >> 1, to = i & 1;
        const int64_t at = b + (to ? j0 + j : mine[j0 + j]);
        page[to][j] = pg_page_of(c, s, at);
        row[to][j] = pg_row_of(c, at);
      }
      if (t == 0) by_moves = pg_div(static_cast<uint32_t>(moves));
      __syncthreads();
      // A warp's items in one line of words, PG_UNROLL x 32 of them in flight: rows of an item in ascending order, items in any.
      const int stride = gridDim.y * PG_WARPS, first = blockIdx.y * PG_WARPS + warp;
      const int row_words = by_words.d, all = first < items ? ((items - first - 1) / stride + 1) * moves * row_words : 0;
      const PgDiv of_moves = by_moves;
      for (int w0 = 0; w0 < all; w0 += 32 * PG_UNROLL) {
        W w[PG_UNROLL];
        char* to[PG_UNROLL];
#pragma unroll
        for (int u = 0; u < PG_UNROLL; ++u) {
          const int i = w0 + lane + 32 * u;
          to[u] = nullptr;
          if (i < all) {
            const int line = static_cast<int>(by_words.of(i)), x = i - line * row_words, turn = static_cast<int>(of_moves.of(line)), j = line - turn * moves;
            const int item = first + turn * stride, rest = item >> 1, layer = static_cast<int>(c.by_head.of(rest)), head = rest - layer * c.heads;
            const PgPool& pool = item & 1 ? c.v : c.k;
            const int p0 = page[0][j], p1 = page[1][j], r0 = row[0][j], r1 = row[1][j];
            char* const p = pool.p + layer * pool.layer + head * pool.head + x * static_cast<int64_t>(sizeof(W));
            if (p0 != p1 || r0 != r1) {
              w[u] = *reinterpret_cast<const W*>(p + p0 * pool.page + r0 * pool.row);
              to[u] = p + p1 * pool.page + r1 * pool.row;
            }
          }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < PG_UNROLL; ++u)
          if (to[u]) *reinterpret_cast<W*>(to[u]) = w[u];
        __syncwarp();
      }
    }
  }
  int32_t* const ticket = c.scratch + at.ticket;
  __syncthreads();
  if (t == 0) {
    __threadfence();
    last = atomicAdd(ticket, 1) == static_cast<int>(gridDim.x * gridDim.y) - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  if (t == 0) *ticket = 0;
  for (int x = t; x < c.slots; x += PG_WARPS * 32) {
    const int wrong = __ldcg(c.scratch + at.mark + x);
    if (wrong) pg_flag(c, wrong);
    else c.lens[x] = static_cast<int>((base ? base[x] : c.lens[x]) + static_cast<int64_t>(kept[x]));
  }
}

// ---------------------------------------------------------------------------------------------- fork
// One cluster of CTAs: new rows of the table go to the scratch first (another slot may still have to read the old ones) and, behind
// the cluster's barrier, into the table; nothing else is waited for. The counts are whole numbers and may change in any order. It is
// as long as four reads that depend on one another: 5 us for four slots, 8 for 64 slots of 128 pages.
constexpr int PG_CLUSTER = 8;
__global__ void __cluster_dims__(PG_CLUSTER, 1, 1) __launch_bounds__(PG_COUNT) pages_fork_kernel(const PgCache c, const int32_t* source, const int32_t* gone) {
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  constexpr int WARPS = PG_CLUSTER * PG_COUNT / 32;
  pg_begin();
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) * PG_CLUSTER + blockIdx.x;
  int32_t *const new_held = c.scratch + at.held, *const new_lens = c.scratch + at.lens, *const rows = c.scratch + at.table;
  // a warp a stretch of 32 entries of a slot's row
  const int stretches = c.max_pages ? (c.max_pages + 31) / 32 : 1;
  const PgDiv by_stretch = pg_div(static_cast<uint32_t>(stretches));
  const int items = c.slots * stretches;  // (fewer than the table's entries and the slots together)
  for (int i = warp; i < items; i += WARPS) {
    const int s = static_cast<int>(by_stretch.of(i)), x = (i - s * stretches) * 32 + lane;
    const int from = source ? source[s] : gone[s] ? -1 : s, old = c.held[s];
    const int64_t mine = static_cast<int64_t>(s) * c.max_pages + x;
    int len = 0, held = -1;  // (-1: the slot stays as it is)
    if (from != s) {
      bool ok = from >= -1 && from < c.slots && old >= 0 && old <= c.max_pages;
      held = 0;
      if (ok && from >= 0) {
        len = c.lens[from];
        held = static_cast<int>(c.by_page.of(static_cast<uint32_t>(max(len, 0))));
        held += held * c.page != len;
        ok = len >= 0 && held <= c.held[from] && held <= c.max_pages;
      }
      if (!ok) {
        if (lane == 0) pg_flag(c, YTC_PAGES_INVALID);
        held = -1;
      } else {
        const int gives = x < old ? c.table[mine] : 0, takes = x < held ? c.table[static_cast<int64_t>(from) * c.max_pages + x] : 0;
        if (x < held) rows[mine] = takes;
        if (x < old && gives >= 0 && gives < c.pages) atomicSub(c.refs + gives, 1);
        if (x < held && takes >= 0 && takes < c.pages) atomicAdd(c.refs + takes, 1);
        if ((x < old && (gives < 0 || gives >= c.pages)) || (x < held && (takes < 0 || takes >= c.pages))) pg_flag(c, YTC_PAGES_INVALID);
      }
    }
    if (x == 0) {
      new_held[s] = held;
      new_lens[s] = len;
    }
  }
  cluster_sync_all();
  for (int i = warp; i < items; i += WARPS) {
    const int s = static_cast<int>(by_stretch.of(i)), x = (i - s * stretches) * 32 + lane;
    const int64_t mine = static_cast<int64_t>(s) * c.max_pages + x;
    const int held = new_held[s], takes = x < c.max_pages ? rows[mine] : 0;
    if (x < held) c.table[mine] = takes;
    if (x == 0 && held >= 0) {
      c.held[s] = held;
      c.lens[s] = new_lens[s];
    }
  }
}

// ---------------------------------------------------------------------------------------------- compact
// One CTA: the new numbers of the pages in use, and what the other cache says of its slots.
__global__ void __launch_bounds__(PG_COUNT) pages_number_kernel(const PgCache c, const PgCache to) {
  pg_begin();
  __shared__ int sums[32];
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  int32_t* const ids = c.scratch + at.ids;
  int32_t* const number = c.scratch + at.number;
  const int t = threadIdx.x;
  const bool wide = reinterpret_cast<uintptr_t>(c.refs) % 16 == 0;
  int found = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 8 * PG_COUNT) {
    const int p = p0 + 8 * t;
    int32_t r[8];
    if (wide && p + 8 <= c.pages) {
      *reinterpret_cast<int4*>(r) = *reinterpret_cast<const int4*>(c.refs + p);
      *reinterpret_cast<int4*>(r + 4) = *reinterpret_cast<const int4*>(c.refs + p + 4);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) r[u] = p + u < c.pages ? c.refs[p + u] : 0;
    }
    int n = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) n += r[u] > 0;
    int total;
    int k = found + pg_scan(n, sums, &total);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (p + u < c.pages) number[p + u] = r[u] > 0 ? k : -1;
      if (r[u] > 0) ids[k++] = p + u;
    }
    found += total;
  }
  __syncthreads();
  const bool full = found > to.pages;
  if (t == 0) {
    c.scratch[at.copies] = full ? -1 : found;
    if (full) pg_flag(to, YTC_PAGES_FULL);
  }
  if (full) return;
  for (int p = t; p < to.pages; p += PG_COUNT) to.refs[p] = p < found ? c.refs[ids[p]] : 0;
  for (int s = t; s < c.slots; s += PG_COUNT) {
    to.lens[s] = c.lens[s];
    to.held[s] = c.held[s];
  }
}
// A warp copies a piece of up to 4 KB of what one page holds of a layer (of a head, where the heads do not lie one behind another). 1.2 GB
// in 384 us, 6.3 TB/s in and out: a plain copy's rate (389 and 402 us with three and four CTAs an SM).
template <int BYTES>
__global__ void __launch_bounds__(PG_WARPS * 32) pages_compact_kernel(const PgCache c, const PgCache to, int row_words, int merged) {
  using W = typename PgWord<BYTES>::type;
  const PgScratch at = pg_scratch(c.slots, c.max_pages, c.pages);
  pg_begin();
  const int pages = c.scratch[at.copies];
  if (pages < 0) return;
  const int64_t entries = static_cast<int64_t>(c.slots) * c.max_pages, threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < entries; i += threads) {
    if (i % c.max_pages >= c.held[i / c.max_pages]) continue;
    const int old = c.table[i];
    const int now = old >= 0 && old < c.pages ? c.scratch[at.number + old] : -1;
    to.table[i] = now;
    if (now < 0) pg_flag(to, YTC_PAGES_INVALID);
  }
  const int blocks = merged ? 1 : c.heads, words = (merged ? c.heads : 1) * c.page * row_words;
  const int rows_a_piece = merged ? 1 : max(1, 32 * PG_UNROLL / row_words);
  const int pieces = merged ? (words + 32 * PG_UNROLL - 1) / (32 * PG_UNROLL) : (c.page + rows_a_piece - 1) / rows_a_piece;
  const int64_t per_page = static_cast<int64_t>(pieces) * blocks * 2 * c.layers;
  const int64_t items = pages * per_page, warps = static_cast<int64_t>(gridDim.x) * PG_WARPS;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * PG_WARPS + (threadIdx.x >> 5); item < items; item += warps) {
    const int now = static_cast<int>(item / per_page);
    int rest = static_cast<int>(item - now * per_page);
    const int piece = rest % pieces;
    rest /= pieces;
    const int head = rest % blocks;
    rest /= blocks;
    const PgPool &x = rest & 1 ? c.v : c.k, &y = rest & 1 ? to.v : to.k;
    const int layer = rest >> 1;
    const char* src = x.p + layer * x.layer + c.scratch[at.ids + now] * x.page + head * x.head;
    char* dst = y.p + layer * y.layer + now * y.page + head * y.head;
    if (merged) {
      const int first = piece * 32 * PG_UNROLL, n = min(32 * PG_UNROLL, words - first);
      pg_copy_rows<W>(dst + first * static_cast<int64_t>(BYTES), n * static_cast<int64_t>(BYTES), src + first * static_cast<int64_t>(BYTES),
                      n * static_cast<int64_t>(BYTES), 1, n);
    } else {
      const int r = piece * rows_a_piece;
      pg_copy_rows<W>(dst + r * y.row, y.row, src + r * x.row, x.row, min(rows_a_piece, c.page - r), row_words);
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
int pg_take(const char* who, const ytcuda_pages* c, PgCache* out) {
  YTC_REQUIRE(c != nullptr, "%s: no cache", who);
  YTC_REQUIRE(c->dtype == YTC_F32 || c->dtype == YTC_BF16 || c->dtype == YTC_F16, "%s: dtype %d is not fp32, bf16 or fp16", who, c->dtype);
  YTC_REQUIRE(c->layers >= 1 && c->pages >= 0 && c->page >= 1 && c->kv_heads >= 1 && c->dim >= 1 && c->slots >= 0 && c->max_pages >= 0,
              "%s: bad extents (layers %d, pages %d of %d positions, heads %d, dim %d, slots %d of %d pages)", who, c->layers, c->pages,
              c->page, c->kv_heads, c->dim, c->slots, c->max_pages);
  // (below them the numbers that kernels keep in 32 bits do not overflow: pieces of all layers of a page, words that a warp moves)
  YTC_REQUIRE(c->page <= 65536 && c->kv_heads <= 65536 && c->dim <= 65536 && c->layers <= 65536 && c->slots < (1 << 30) && c->pages < (1 << 30) &&
                  static_cast<int64_t>(c->slots) * c->max_pages < (1ll << 31) &&
                  static_cast<int64_t>(c->page) * c->kv_heads * c->dim < (1ll << 31) &&
                  static_cast<int64_t>(c->layers) * c->kv_heads * c->dim <= (1ll << 25) &&
                  static_cast<int64_t>(c->layers) * c->kv_heads * c->dim * c->page < (1ll << 36),
              "%s: extents above the limits (pages of 65536 positions and 2^31 elements a layer, 2^25 elements a position and 2^36 a page of all "
              "layers, 2^30 slots and pages, tables of 2^31 entries)",
              who);
  YTC_REQUIRE(c->slots == 0 || c->pages == 0 || (c->k && c->v && c->lens && c->held && c->refs && c->status && c->scratch &&
                                                (c->table || c->max_pages == 0)),
              "%s: null tensor in the cache", who);
  const int size = dtype_size(c->dtype);
  YTC_REQUIRE((reinterpret_cast<uint64_t>(c->k) | reinterpret_cast<uint64_t>(c->v)) % size == 0, "%s: misaligned pool", who);
  // (the stride of an axis of one element says nothing: it must not decide how rows are copied)
  auto pool = [&](void* p, const int64_t* s) {
    const int64_t any = static_cast<int64_t>(c->dim) * size;
    return PgPool{static_cast<char*>(p), c->layers == 1 ? any : s[0] * size, c->pages == 1 ? any : s[1] * size,
                  c->kv_heads == 1 ? any : s[2] * size, c->page == 1 ? any : s[3] * size};
  };
  for (int i = 0; i < 4; ++i) YTC_REQUIRE(c->k_strides[i] >= 0 && c->v_strides[i] >= 0, "%s: negative stride in a pool", who);
  *out = PgCache{pool(c->k, c->k_strides), pool(c->v, c->v_strides), pg_div(static_cast<uint32_t>(c->page)),
                 pg_div(static_cast<uint32_t>(c->kv_heads)), c->table, c->lens, c->held, c->refs, c->status, c->scratch,
                 c->layers, c->pages, c->page, c->kv_heads, c->dim, c->slots, c->max_pages};
  return YTC_OK;
}

int pg_rows(const char* who, const char* what, const void* p, const int64_t* strides, int size, PgRows* out) {
  YTC_REQUIRE(p && strides, "%s: null %s", who, what);
  YTC_REQUIRE(reinterpret_cast<uint64_t>(p) % size == 0, "%s: misaligned %s", who, what);
  *out = PgRows{const_cast<char*>(static_cast<const char*>(p)), strides[0] * size, strides[1] * size};
  return YTC_OK;
}

// Two boxes meet where a sum of strides, each times a number of its range (an index of a minus one of b), is the distance of their first
// elements. The strides are tried from the largest down, those numbers only that the smaller ones can make up for: one or two for strides
// of axes that lie in one another. Where that takes too long they count as meeting.
struct PgMeet {
  int64_t stride[9], lo[9], hi[9], least[10], most[10];  // least, most: of all terms from one on
  int n, left;
  bool from(int i, int64_t rest) {
    if (rest < least[i] || rest > most[i]) return false;
    if (i == n || (stride[i] == 1 && i == n - 1)) return true;
    if (--left < 0) return true;
    // stride x in rest - most .. rest - least of the others
    const auto down = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    const int64_t first = -down(most[i + 1] - rest, stride[i]), last = down(rest - least[i + 1], stride[i]);
    for (int64_t x = first > lo[i] ? first : lo[i]; x <= last && x <= hi[i]; ++x)
      if (from(i + 1, rest - x * stride[i])) return true;
    return false;
  }
};
bool pg_meet(const PgBox& a, const PgBox& b, int size) {
  if (!a.p || !b.p) return false;
  PgMeet m;
  m.n = 0;
  m.left = 100000;
  const auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    if (stride < 0) {
      const int64_t x = lo;
      stride = -stride, lo = -hi, hi = -x;
    }
    if (stride == 0 || lo == hi) return;
    int i = 0;
    while (i < m.n && m.stride[i] > stride) ++i;
    if (i < m.n && m.stride[i] == stride) {
      m.lo[i] += lo, m.hi[i] += hi;
      return;
    }
    for (int j = m.n++; j > i; --j) m.stride[j] = m.stride[j - 1], m.lo[j] = m.lo[j - 1], m.hi[j] = m.hi[j - 1];
    m.stride[i] = stride, m.lo[i] = lo, m.hi[i] = hi;
  };
  for (int i = 0; i < 4; ++i) {
    if (a.extent[i] <= 0 || b.extent[i] <= 0) return false;
    add(a.stride[i] / size, 0, a.extent[i] - 1);
    add(b.stride[i] / size, -(b.extent[i] - 1), 0);
  }
  add(1, -(b.dim - 1), a.dim - 1);
  m.least[m.n] = m.most[m.n] = 0;
  for (int i = m.n - 1; i >= 0; --i) m.least[i] = m.least[i + 1] + m.stride[i] * m.lo[i], m.most[i] = m.most[i + 1] + m.stride[i] * m.hi[i];
  return m.from(0, (b.p - a.p) / size);
}

static unsigned copy_grid(int64_t items) {
  const int64_t blocks = (items + PG_WARPS - 1) / PG_WARPS, most = 8ll * sm_count();
  return static_cast<unsigned>(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

}  // namespace ytk

using namespace ytk;

// One launch for each width in which rows can be copied.
#define PG_BY_WIDTH(width, launch)    \
  do {                                \
    if ((width) == 16) {              \
      constexpr int B = 16;           \
      launch;                         \
    } else if ((width) == 4) {        \
      constexpr int B = 4;            \
      launch;                         \
    } else {                          \
      constexpr int B = 2;            \
      launch;                         \
    }                                 \
  } while (0)

extern "C" {

uint64_t ytcuda_pages_scratch(const ytcuda_pages* cache) {
  if (!cache || cache->slots < 0 || cache->max_pages < 0 || cache->pages < 0) return 0;
  return 4ull * static_cast<uint64_t>(pg_scratch(cache->slots, cache->max_pages, cache->pages).words);
}

int ytcuda_pages_append(const ytcuda_pages* cache, int layer, const void* k, const void* v, const int64_t* strides,
                        const int32_t* starts, int rows, void* stream) {
  const char* who = "ytcuda_pages_append";
  PgCache c;
  if (const int rc = pg_take(who, cache, &c)) return rc;
  YTC_REQUIRE(layer >= 0 && layer < c.layers, "%s: layer %d of %d", who, layer, c.layers);
  YTC_REQUIRE(rows >= 0, "%s: negative number of rows", who);
  if (rows == 0 || c.slots == 0) return YTC_OK;
  YTC_REQUIRE(starts && strides, "%s: null starts or strides", who);
  YTC_REQUIRE(c.pages > 0, "%s: a pool without pages", who);
  const int size = dtype_size(cache->dtype);
  PgRows kr, vr;
  if (const int rc = pg_rows(who, "k", k, strides, size, &kr)) return rc;
  if (const int rc = pg_rows(who, "v", v, strides + 2, size, &vr)) return rc;
  const int width = pg_width(pg_bits(c.k) | pg_bits(c.v) | pg_bits(kr) | pg_bits(vr) | static_cast<uint64_t>(c.dim * size));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int words = c.dim * size / width, a_round = 32 * PG_UNROLL / words, run = a_round < 1 ? 1 : a_round > 32 ? 32 : a_round;
  const int64_t items = (static_cast<int64_t>(rows) + run - 1) / run * 2 * c.heads;
  const PgDiv by_words = pg_div(static_cast<uint32_t>(words));
  YTC_REQUIRE(items < (1ll << 30), "%s: %d rows of %d heads are too many", who, rows, c.heads);
  PG_BY_WIDTH(width, YTC_CUDA(pg_launch(pages_append_kernel<B>, dim3(copy_grid(items)), dim3(PG_WARPS * 32), 0, st, c, kr, vr, starts, rows, layer,
                                        by_words, run)));
  count_launch();
  return YTC_OK;
}

int ytcuda_pages_reserve(const ytcuda_pages* cache, const int32_t* counts, void* stream) {
  const char* who = "ytcuda_pages_reserve";
  PgCache c;
  if (const int rc = pg_take(who, cache, &c)) return rc;
  if (c.slots == 0) return YTC_OK;
  YTC_REQUIRE(counts != nullptr, "%s: null counts", who);
  YTC_REQUIRE(c.pages > 0, "%s: a pool without pages", who);
  const int size = dtype_size(cache->dtype);
  const int width = pg_width(pg_bits(c.k) | pg_bits(c.v) | static_cast<uint64_t>(c.dim * size));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  YTC_CUDA(pg_launch(pages_reserve_kernel, dim3(1), dim3(PG_COUNT), 0, st, c, counts));
  count_launch();
  const int rows_a_piece = 32 * PG_UNROLL * width / (c.dim * size);
  const unsigned grid = copy_grid(2ll * c.slots * c.layers * c.heads * (rows_a_piece > 1 ? (c.page + rows_a_piece - 1) / rows_a_piece : c.page));
  PG_BY_WIDTH(width, YTC_CUDA(pg_launch(pages_copy_kernel<B>, dim3(grid), dim3(PG_WARPS * 32), 0, st, c, c.dim * size / B)));
  count_launch();
  return YTC_OK;
}

int ytcuda_pages_keep(const ytcuda_pages* cache, const int32_t* kept, const int32_t* accepted, int depth, const int32_t* base,
                      void* stream) {
  const char* who = "ytcuda_pages_keep";
  PgCache c;
  if (const int rc = pg_take(who, cache, &c)) return rc;
  YTC_REQUIRE(depth >= 0, "%s: negative depth", who);
  if (c.slots == 0) return YTC_OK;
  YTC_REQUIRE(kept != nullptr, "%s: null kept", who);
  YTC_REQUIRE(c.pages > 0, "%s: a pool without pages", who);
  const int size = dtype_size(cache->dtype);
  const int width = pg_width(pg_bits(c.k) | pg_bits(c.v) | static_cast<uint64_t>(c.dim * size));
  // three CTAs an SM, all that it holds, where there is that much to move: a warp's items one behind another
  const int64_t a_slot = (2ll * c.layers * c.heads + PG_WARPS - 1) / PG_WARPS, most = (3ll * sm_count() + c.slots - 1) / c.slots;
  const dim3 grid(static_cast<unsigned>(c.slots), accepted ? static_cast<unsigned>(a_slot < most ? a_slot : most) : 1u);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const PgDiv by_words = pg_div(static_cast<uint32_t>(c.dim * size / width));
  PG_BY_WIDTH(width, YTC_CUDA(pg_launch(pages_keep_kernel<B>, grid, dim3(PG_WARPS * 32), 0, st, c, kept, accepted, depth, base, by_words)));
  count_launch();
  return YTC_OK;
}

int ytcuda_pages_fork(const ytcuda_pages* cache, const int32_t* source, const int32_t* gone, void* stream) {
  const char* who = "ytcuda_pages_fork";
  PgCache c;
  if (const int rc = pg_take(who, cache, &c)) return rc;
  if (c.slots == 0) return YTC_OK;
  YTC_REQUIRE((source != nullptr) != (gone != nullptr), "%s: source or gone, one of them", who);
  YTC_REQUIRE(c.pages > 0, "%s: a pool without pages", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  YTC_CUDA(pg_launch(pages_fork_kernel, dim3(PG_CLUSTER), dim3(PG_COUNT), 0, st, c, source, gone));
  count_launch();
  return YTC_OK;
}

int ytcuda_pages_compact(const ytcuda_pages* cache, const ytcuda_pages* into, void* stream) {
  const char* who = "ytcuda_pages_compact";
  PgCache c, to;
  if (const int rc = pg_take(who, cache, &c)) return rc;
  if (const int rc = pg_take(who, into, &to)) return rc;
  YTC_REQUIRE(cache->dtype == into->dtype && c.layers == to.layers && c.page == to.page && c.heads == to.heads && c.dim == to.dim &&
                  c.slots == to.slots && c.max_pages == to.max_pages,
              "%s: the caches differ in type, layers, page, heads, dim, slots or table", who);
  if (c.slots == 0) return YTC_OK;
  YTC_REQUIRE(c.pages > 0 && to.pages > 0, "%s: a pool without pages", who);
  const int size = dtype_size(cache->dtype);
  for (const PgPool* x : {&c.k, &c.v})
    for (const PgPool* y : {&to.k, &to.v})
      YTC_REQUIRE(!pg_meet(pg_box(*x, c), pg_box(*y, to), size), "%s: the pools of the caches share memory", who);
  const auto ints = [](const PgCache& x, int i) {
    const int64_t n[4] = {static_cast<int64_t>(x.slots) * x.max_pages, x.slots, x.slots, x.pages};
    const int32_t* const p[4] = {x.table, x.lens, x.held, x.refs};
    return PgBox{reinterpret_cast<const char*>(p[i]), {n[i] > 0, 1, 1, 1}, {0, 0, 0, 0}, n[i]};
  };
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) YTC_REQUIRE(!pg_meet(ints(c, i), ints(to, j), 4), "%s: the tables or counts of the caches share memory", who);
  const int width = pg_width(pg_bits(c.k) | pg_bits(c.v) | pg_bits(to.k) | pg_bits(to.v) | static_cast<uint64_t>(c.dim * size));
  int merged = 1;
  for (const PgPool* p : {&c.k, &c.v, &to.k, &to.v})
    merged = merged && p->row == c.dim * size && (p->head == c.page * p->row || c.heads == 1);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  YTC_CUDA(pg_launch(pages_number_kernel, dim3(1), dim3(PG_COUNT), 0, st, c, to));
  count_launch();
  const unsigned grid = copy_grid(1ll << 30);
  PG_BY_WIDTH(width, YTC_CUDA(pg_launch(pages_compact_kernel<B>, dim3(grid), dim3(PG_WARPS * 32), 0, st, c, to, c.dim * size / B, merged)));
  count_launch();
  return YTC_OK;
}

}  // extern "C"
