// Attention of new rows (single tokens, chains, trees of drafted tokens) over a cache in pages.
//
// Of one slot and key head the rows are (node, query head of the group), node by node, in tiles of RT; a unit is such a tile with
// all keys of its slot, in tiles of BN positions. All units' key tiles in one line are cut into equal shares, one for each CTA,
// wherever the cuts fall: ragged lengths cost nothing, and a single long sequence still uses every SM. A unit that a cut runs
// through leaves sums (O, m, l) of each piece in the workspace, which a second launch joins in the order of the pieces. Lengths
// and starts are read on the device; the host knows neither.
//
// With s = scale q.k over the seen positions: m = max s, l = sum exp(s - m), o = sum exp(s - m) v / l, in one pass over the keys
// with the running maximum; 2 to the power of s log2(e) throughout. A cut's pieces join as m = max m_i, O = sum 2^(m_i - m) O_i.
#include <math_constants.h>

#include <type_traits>

#include "pages.cuh"
#include "ptx_sm100.cuh"

namespace ytk {

constexpr int PA_THREADS = 128;
constexpr int PA_TREE = 1024;  // most nodes of a tree
constexpr float PA_LOG2E = 1.4426950408889634f;

struct PaParams {
  PgCache c;  // (the pools at the layer)
  PgRows q, k, v, o;
  PgDiv by_group;  // division by the query heads of a key head
  const int32_t *starts, *parents;
  int rows, groups;
  int fresh;    // k and v hold the new rows: they are read from there, and stored
  int wide, words;  // rows in pieces of 16 bytes (else of an element), their number
  float scale;  // times log2(e)
  float* work;  // pieces of cut units
  int4* cuts;   // two words for each CTA: the unit that goes on behind its share
  int* timeout; // the device's status word
  int box;      // rows of a page that a TMA copy takes (0: none)
};

// What a slot brings: its rows in the call, its nodes, its length.
struct PaSlot {
  int start, nodes, len;
};
__device__ __forceinline__ PaSlot pa_slot(const PaParams& p, int s, bool* bad) {
  PaSlot r{p.starts[s], p.starts[s + 1], p.c.lens[s]};
  const int end = r.nodes, held = p.c.held[s];
  r.nodes = end - r.start;
  const bool ok = r.start >= 0 && end >= r.start && end <= p.rows && r.len >= 0 && !(p.parents && r.nodes > PA_TREE) &&
                  r.len <= 0x7ffffff0 - r.nodes && held <= p.c.max_pages &&
                  r.len + static_cast<int64_t>(p.fresh ? 0 : r.nodes) <= static_cast<int64_t>(held) * p.c.page;
  if (!ok) {
    *bad = *bad || r.nodes != 0;
    r.nodes = 0;
  }
  return r;
}
// The units of a slot are its heads' row tiles, the row tiles of a head next to one another (they read the same keys at about the same
// time). Work is counted in costs of key tiles: a unit of up to RW rows costs ONE a key tile, one of two such blocks (RT = 2 RW) costs
// BOTH, less than twice as much, since it reads the keys once. All numbers stay below 2^31: the host sees to that.
template <int RT, int RW>
struct PaCost {
  static_assert(RT == RW || RT == 2 * RW, "one block of rows or two");
  static constexpr uint32_t BLOCKS = RT / RW, ONE = BLOCKS == 1 ? 1 : 2, BOTH = BLOCKS == 1 ? 1 : 3;
  static __device__ __forceinline__ uint32_t of(uint32_t blocks) { return BLOCKS == 1 ? blocks : blocks / 2 * BOTH + blocks % 2 * ONE; }
};
template <int BN>
__device__ __forceinline__ uint32_t pa_key_tiles(const PaSlot& s) {
  return (static_cast<uint32_t>(s.len) + static_cast<uint32_t>(s.nodes) + BN - 1) / BN;
}
template <int RW>
__device__ __forceinline__ uint32_t pa_row_blocks(const PaParams& p, const PaSlot& s) {
  return (static_cast<uint32_t>(s.nodes) * static_cast<uint32_t>(p.groups) + RW - 1) / RW;
}
template <int RT, int RW, int BN>
__device__ __forceinline__ uint32_t pa_work(const PaParams& p, const PaSlot& s) {
  return s.nodes ? pa_key_tiles<BN>(s) * PaCost<RT, RW>::of(pa_row_blocks<RW>(p, s)) * p.c.heads : 0u;
}

// The share of a CTA: from .. to of all costs, the first of them number `off` of slot `slot`. Shares differ by at most one, the longer
// ones first: share i begins at i * each + min(i, more). No share is shorter than a key tile of a unit.
struct PaShare {
  uint32_t from, to, off, each, more;
  int slot;
};
__device__ __forceinline__ uint32_t pa_share_of(const PaShare& s, uint32_t at) {
  const uint32_t longer = s.more * (s.each + 1);
  return at < longer ? at / (s.each + 1) : s.more + (at - longer) / s.each;
}
// All threads of the CTA call it; one warp works it out.
template <int RT, int RW, int BN>
__device__ __forceinline__ void pa_share(const PaParams& p, PaShare* out) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    bool bad = false, down = false;
    uint32_t total = 0, w = 0;
    for (int s0 = 0; s0 < p.c.slots; s0 += 32) {
      w = s0 + lane < p.c.slots ? pa_work<RT, RW, BN>(p, pa_slot(p, s0 + lane, &bad)) : 0;
      down = down || (s0 + lane < p.c.slots && p.starts[s0 + lane + 1] < p.starts[s0 + lane]);
      total += __reduce_add_sync(0xffffffffu, w);
    }
    // (starts that descend: slots would claim the same rows, and the sum of their costs could pass 32 bits. Nothing is computed.)
    if (__any_sync(0xffffffffu, down)) total = 0;
    if (blockIdx.x == 0 && __any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.c.status, YTC_PAGES_INVALID);
    PaShare r;
    const uint32_t parts = min(gridDim.x, max(1u, total / PaCost<RT, RW>::BOTH));
    r.each = total / parts;
    r.more = total - r.each * parts;
    r.from = min(total, blockIdx.x * r.each + min(blockIdx.x, r.more));
    r.to = blockIdx.x < parts ? r.from + r.each + (blockIdx.x < r.more) : r.from;
    r.off = 0;
    r.slot = p.c.slots;
    uint32_t before = 0;
    for (int s0 = 0; s0 < p.c.slots; s0 += 32) {
      if (p.c.slots > 32) w = s0 + lane < p.c.slots ? pa_work<RT, RW, BN>(p, pa_slot(p, s0 + lane, &bad)) : 0;
      uint32_t x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + x > r.from);
      if (hit) {
        const int l = __ffs(hit) - 1;
        r.slot = s0 + l;
        r.off = r.from - before - __shfl_sync(0xffffffffu, x - w, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) *out = r;
  }
  __syncthreads();
}

// A piece of work: key tiles t0 .. t1 of a unit that sees `tiles` of them, each of cost `weight`, the first of them number `first` of all costs.
struct PaPart {
  PaSlot s;
  uint32_t tiles, t0, t1, weight, first;
  int slot, head, rtile, row0, rows, rows_all;
};
// Where a CTA is in its share.
struct PaAt {
  uint32_t pos, end, off;
  int slot;
  __device__ __forceinline__ explicit PaAt(const PaShare& s) : pos(s.from), end(s.to), off(s.off), slot(s.slot) {}
};
// The next piece of the share; false behind the last one. A key tile belongs to the share that its first cost lies in. No node sees a
// later one: tiles behind the last node of a row tile are passed over. In the line they count all the same, but the row tiles stand
// there as first, last, second, last but one, ..., so that what is passed over is about the same in every share of many row tiles (four
// prompts of 8000, fp16, 8 key heads of 4: 9.2 ms with all tiles, 8.6 passed over in order, 5.1 so; 3.2, 655 TFLOP/s, since tiles that
// all rows see are neither masked nor looked through).
template <int RT, int RW, int BN>
__device__ __forceinline__ bool pa_next(const PaParams& p, PaAt* at, PaPart* out) {
  using Cost = PaCost<RT, RW>;
  while (at->pos < at->end) {
    bool bad = false;
    PaPart& r = *out;
    r.s = pa_slot(p, at->slot, &bad);
    const uint32_t work = pa_work<RT, RW, BN>(p, r.s);
    if (at->off >= work) {  // (slots without rows too)
      at->off -= work;
      ++at->slot;
      continue;
    }
    r.slot = at->slot;
    const uint32_t tiles = pa_key_tiles<BN>(r.s), blocks = pa_row_blocks<RW>(p, r.s), a_head = tiles * Cost::of(blocks);
    const uint32_t head = at->off / a_head, in_head = at->off - head * a_head;
    const uint32_t unit = in_head / (tiles * Cost::BOTH), in_unit = in_head - unit * (tiles * Cost::BOTH);
    const uint32_t full = blocks / Cost::BLOCKS;  // units of BOTH
    r.weight = unit < full ? Cost::BOTH : Cost::ONE;
    const uint32_t n = min(tiles * r.weight - in_unit, at->end - at->pos);
    r.first = at->pos - in_unit;
    r.t0 = (in_unit + r.weight - 1) / r.weight;
    r.t1 = (in_unit + n + r.weight - 1) / r.weight;
    at->pos += n;
    at->off += n;
    r.head = static_cast<int>(head);
    r.rtile = static_cast<int>(unit >= full ? unit : unit & 1 ? full - 1 - unit / 2 : unit / 2);
    r.row0 = r.rtile * RT;
    r.rows_all = r.s.nodes * p.groups;
    r.rows = min(RT, r.rows_all - r.row0);
    const uint32_t last = p.by_group.of(static_cast<uint32_t>(r.row0 + r.rows - 1));  // node of the last row
    r.tiles = (static_cast<uint32_t>(r.s.len) + last + BN) / BN;
    r.t1 = min(r.t1, r.tiles);
    if (r.t0 >= r.t1) continue;
    return true;
  }
  return false;
}

// Floats of a piece in the workspace: O [rt][dp], m [rt], l [rt]. A CTA has two: its first and its last unit may be cut.
__host__ __device__ __forceinline__ int64_t pa_piece(int rt, int dp) { return static_cast<int64_t>(rt) * (dp + 2); }
template <int RT, int DP>
__device__ __forceinline__ float* pa_piece_of(const PaParams& p, const PaPart& w) {
  return p.work + (2 * static_cast<int64_t>(blockIdx.x) + (w.t0 == 0)) * pa_piece(RT, DP);
}
// What joining has to know of the unit that goes on behind this CTA's share: rows (0: no such unit), first row, head, start of the
// slot's rows; first and last share. Written by one thread.
struct PaCut {
  int4* at;  // null: not this thread
  __device__ __forceinline__ PaCut(const PaParams& p, bool mine) : at(mine ? p.cuts + 2 * blockIdx.x : nullptr) {
    if (mine) at[0] = make_int4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void note(const PaShare& sh, const PaPart& w) const {
    if (at && w.t1 < w.tiles) {
      at[0] = make_int4(w.rows, w.row0, w.head, w.s.start);
      at[1] = make_int4(static_cast<int>(pa_share_of(sh, w.first)), static_cast<int>(pa_share_of(sh, w.first + (w.tiles - 1) * w.weight)), 0, 0);
    }
  }
};
// Where the result of a row goes.
__device__ __forceinline__ char* pa_out(const PaParams& p, int start, int head, int row) {
  const int node = static_cast<int>(p.by_group.of(row)), g = row - node * p.groups;
  return p.o.p + (start + static_cast<int64_t>(node)) * p.o.row + static_cast<int64_t>(head * p.groups + g) * p.o.head;
}
__device__ __forceinline__ const char* pa_query(const PaParams& p, const PaPart& w, int row) {
  const int node = static_cast<int>(p.by_group.of(row)), g = row - node * p.groups;
  return p.q.p + (w.s.start + static_cast<int64_t>(node)) * p.q.row + static_cast<int64_t>(w.head * p.groups + g) * p.q.head;
}

// Element loads and stores in the cache's type; 16-bit results round to nearest even.
__device__ __forceinline__ float pa_load(const float* p) { return *p; }
__device__ __forceinline__ float pa_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float pa_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void pa_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void pa_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void pa_store(__half* p, float v) { *p = __float2half_rn(v); }

// Ancestors of the nodes of a row tile: bit j of seen[i - first] says that node j is node i or one of its ancestors. `up` takes
// the slot's parents. All threads of the CTA; a parent that is none counts as -1.
__device__ __forceinline__ void pa_ancestors(const PaParams& p, const PaSlot& s, int first, int count, uint32_t (*seen)[PA_TREE / 32 + 1],
                                             int16_t* up) {
  const int t = threadIdx.x, nt = blockDim.x;
  for (int i = t; i < s.nodes; i += nt) {
    int a = p.parents[s.start + i];
    if (a < -1 || a >= i) {
      atomicOr(p.c.status, YTC_PAGES_INVALID);
      a = -1;
    }
    up[i] = static_cast<int16_t>(a);
  }
  const int words = (s.nodes + 31) / 32;
  for (int i = t; i < count * words; i += nt) seen[i / words][i % words] = 0;
  __syncthreads();
  for (int i = t; i < count && first + i < s.nodes; i += nt)
    for (int j = first + i; j >= 0; j = up[j]) seen[i][j >> 5] |= 1u << (j & 31);
  __syncthreads();
}

// Which of 64 keys a node sees, the first of them being node n0 of its slot (negative: in front of the nodes). line: its ancestors
// (nullptr: a chain).
__device__ __forceinline__ uint64_t pa_sees(const uint32_t* line, int words, int node, int n0) {
  const int upto = line ? -n0 : node + 1 - n0;  // keys that are seen whatever the tree
  const uint64_t low = upto >= 64 ? ~0ull : upto > 0 ? (1ull << upto) - 1 : 0ull;
  if (!line || upto >= 64) return low;
  const int first = n0 > 0 ? n0 >> 5 : 0, shift = n0 > 0 ? n0 & 31 : 0;
  uint32_t w[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) w[i] = first + i < words ? line[first + i] : 0u;
  const uint64_t bits = static_cast<uint64_t>(__funnelshift_r(w[0], w[1], shift)) |
                        static_cast<uint64_t>(__funnelshift_r(w[1], w[2], shift)) << 32;
  return low | (n0 < 0 ? bits << -n0 : bits);
}

// Whether any of NK keys is hidden from any row of the warp: in a prompt's tiles few are, and looking for hidden values that are not
// finite takes as long as the products.
template <int NK>
__device__ __forceinline__ bool pa_any_hidden(const uint64_t (&sees)[2]) {
  constexpr uint64_t all = NK < 64 ? (1ull << (NK % 64)) - 1 : ~0ull;
  return __any_sync(0xffffffffu, (sees[0] & sees[1] & all) != all);
}

// Positions of a slot whose rows are in the pages.
__device__ __forceinline__ uint32_t pa_paged(const PaParams& p, const PaPart& w) {
  return static_cast<uint32_t>(w.s.len) + (p.fresh ? 0u : static_cast<uint32_t>(w.s.nodes));
}
// What the table says of a position, as it stands there: it is asked for ahead of its use, and a warp that looks at a number waits for
// it. pa_checked: the page, -1 where there is none (which is noted).
__device__ __forceinline__ int pa_lookup(const PaParams& p, const PaPart& w, uint32_t at) {
  int pg = -1;
  const int i = static_cast<int>(p.c.by_page.of(at));
  if (at < pa_paged(p, w) && i < p.c.held[w.slot] && i < p.c.max_pages) pg = p.c.table[static_cast<int64_t>(w.slot) * p.c.max_pages + i];
  return pg;
}
__device__ __forceinline__ int pa_checked(const PaParams& p, int pg) {
  if (pg >= 0 && pg < p.c.pages) return pg;
  atomicOr(p.c.status, YTC_PAGES_INVALID);
  return -1;
}
// Where the rows of a position of a slot and head lie; nullptr where there are none. `pg`: what the table says of it.
struct PaRow {
  const char *k, *v;
};
__device__ __forceinline__ PaRow pa_row(const PaParams& p, const PaPart& w, uint32_t at, int pg) {
  PaRow r{nullptr, nullptr};
  const uint32_t len = w.s.len;
  if (at < pa_paged(p, w)) {
    pg = pa_checked(p, pg);
    if (pg < 0) return r;
    const int row = pg_row_of(p.c, at);
    r.k = p.c.k.p + pg * p.c.k.page + w.head * p.c.k.head + row * p.c.k.row;
    r.v = p.c.v.p + pg * p.c.v.page + w.head * p.c.v.head + row * p.c.v.row;
  } else if (at - len < static_cast<uint32_t>(w.s.nodes)) {
    const int64_t row = w.s.start + static_cast<int64_t>(at - len);
    r.k = p.k.p + row * p.k.row + w.head * p.k.head;
    r.v = p.v.p + row * p.v.row + w.head * p.v.head;
  }
  return r;
}

__device__ __forceinline__ void pa_copy16(uint32_t dst, const char* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pa_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pa_copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------------------------- FFMA form
// Rows that are not whole 16-byte words on their boundaries (odd dims and strides), element by element. 8 x 16 threads: thread
// (a, b) holds rows a + 8 i (RPT of them) with keys b + 16 j of S and with columns 4 b + 64 j of O. Two tiles of keys and values as
// fp32 in shared memory: the next one is read before one is worked on. Bound by the loads, an element each: dim 100 in fp16, one token and
// four heads a group behind 4000 keys, eight slots, 710 us, 0.14 TB/s.
template <typename T, int DP, int RPT>
struct PaFfma {
  static constexpr int RT = 8 * RPT, BN = DP == 64 ? 64 : 32;
  float q[RT][DP + 4], k[2][BN][DP + 4], v[2][BN][DP], s[RT][BN + 4];
  const T* row[2][2][BN];
  uint32_t seen[RT][PA_TREE / 32 + 1];
  int16_t up[PA_TREE];
  PaShare share;
};

// O += S V of one tile. HIDDEN: weights of zero take nothing along (a hidden position holds an infinity or NaN, and 0 x infinity
// would spoil every row).
template <int DP, int RPT, int BN, bool HIDDEN>
__device__ __forceinline__ void pa_ffma_values(const float (*s)[BN + 4], const float (*v)[DP], int a, int b, float (*o)[DP / 16]) {
#pragma unroll(HIDDEN ? 1 : 2)
  for (int kk = 0; kk < BN; kk += 4) {
    float4 e[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) e[i] = *reinterpret_cast<const float4*>(&s[a + 8 * i][kk]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) {
        const float4 y = *reinterpret_cast<const float4*>(&v[kk + u][4 * b + 64 * j]);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float w = u == 0 ? e[i].x : u == 1 ? e[i].y : u == 2 ? e[i].z : e[i].w;
          if (HIDDEN && w == 0.f) continue;
          o[i][4 * j] = fmaf(w, y.x, o[i][4 * j]);
          o[i][4 * j + 1] = fmaf(w, y.y, o[i][4 * j + 1]);
          o[i][4 * j + 2] = fmaf(w, y.z, o[i][4 * j + 2]);
          o[i][4 * j + 3] = fmaf(w, y.w, o[i][4 * j + 3]);
        }
      }
  }
}

template <typename T, int DP, int RPT>
__global__ void __launch_bounds__(PA_THREADS) paged_attn_ffma_kernel(const PaParams p) {
  using S = PaFfma<T, DP, RPT>;
  constexpr int RT = S::RT, BN = S::BN, KPT = BN / 16, CJ = DP / 64;
  extern __shared__ __align__(128) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  pg_begin();
  const int t = threadIdx.x, a = t >> 4, b = t & 15;
  const PgCache& c = p.c;
  pa_share<RT, RT, BN>(p, &sm.share);
  const PaCut cut(p, threadIdx.x == 0);
  PaAt at(sm.share);
  PaPart w;
  while (pa_next<RT, RT, BN>(p, &at, &w)) {
    const int nodes = w.s.nodes, words = (nodes + 31) / 32;
    const int node0 = static_cast<int>(p.by_group.of(w.row0)), node1 = static_cast<int>(p.by_group.of(w.row0 + w.rows - 1));
    // Thread t < BN finds where row t of a tile lies, with the page that it looked up one tile earlier.
    int pg = t < BN ? pa_lookup(p, w, w.t0 * BN + t) : -1;
    const auto find = [&](uint32_t tile) {
      if (t < BN && tile < w.t1) {
        const PaRow r = pa_row(p, w, tile * BN + t, pg);
        sm.row[tile & 1][0][t] = reinterpret_cast<const T*>(r.k);
        sm.row[tile & 1][1][t] = reinterpret_cast<const T*>(r.v);
        if (tile + 1 < w.t1) pg = pa_lookup(p, w, (tile + 1) * BN + t);
      }
    };
    const auto fetch = [&](uint32_t tile) {
      if (tile >= w.t1) return;
      const int x = tile & 1;
#pragma unroll 4
      for (int i = t; i < BN * DP; i += PA_THREADS) {
        const int r = i / DP, d = i % DP;
        const T *kp = sm.row[x][0][r], *vp = sm.row[x][1][r];
        const bool there = kp != nullptr && d < c.dim;
        sm.k[x][r][d] = there ? pa_load(kp + d) : 0.f;
        sm.v[x][r][d] = there ? pa_load(vp + d) : 0.f;
      }
    };
    __syncthreads();  // (the part before is done with the shared memory)
    find(w.t0);
    find(w.t0 + 1);
    __syncthreads();
    fetch(w.t0);
    for (int i = t; i < RT * DP; i += PA_THREADS) {
      const int r = i / DP, d = i % DP;
      sm.q[r][d] = r < w.rows && d < c.dim ? pa_load(reinterpret_cast<const T*>(pa_query(p, w, w.row0 + r)) + d) * p.scale : 0.f;
    }
    if (p.parents && static_cast<uint64_t>(w.t1) * BN > static_cast<uint32_t>(w.s.len)) pa_ancestors(p, w.s, node0, node1 - node0 + 1, sm.seen, sm.up);
    float m[RPT], l[RPT], o[RPT][4 * CJ];
    int node[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      m[i] = -CUDART_INF_F;
      l[i] = 0.f;
      node[i] = static_cast<int>(p.by_group.of(w.row0 + min(a + 8 * i, w.rows - 1)));
#pragma unroll
      for (int j = 0; j < 4 * CJ; ++j) o[i][j] = 0.f;
    }
#pragma unroll 1
    for (uint32_t tile = w.t0; tile < w.t1; ++tile) {
      __syncthreads();
      fetch(tile + 1);
      find(tile + 2);
      const int cur = tile & 1, n0 = static_cast<int>(tile * BN) - w.s.len;  // the node at the tile's first key
      float x[RPT][KPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < KPT; ++j) x[i][j] = 0.f;
#pragma unroll 4
      for (int d = 0; d < DP; d += 4) {
        float4 kk[KPT];
#pragma unroll
        for (int j = 0; j < KPT; ++j) kk[j] = *reinterpret_cast<const float4*>(&sm.k[cur][b + 16 * j][d]);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(&sm.q[a + 8 * i][d]);
#pragma unroll
          for (int j = 0; j < KPT; ++j)
            x[i][j] = fmaf(qq.x, kk[j].x, fmaf(qq.y, kk[j].y, fmaf(qq.z, kk[j].z, fmaf(qq.w, kk[j].w, x[i][j]))));
        }
      }
      const bool masked = n0 + BN > 0;
      if (masked) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const uint64_t sees = pa_sees(p.parents ? sm.seen[node[i] - node0] : nullptr, words, node[i], n0);
#pragma unroll
          for (int j = 0; j < KPT; ++j)
            if (!((sees >> (b + 16 * j)) & 1)) x[i][j] = -CUDART_INF_F;
        }
      }
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        float top = m[i];
#pragma unroll
        for (int j = 0; j < KPT; ++j) top = fmaxf(top, x[i][j]);
#pragma unroll
        for (int k = 8; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float ref = top == -CUDART_INF_F ? 0.f : top, shrink = exp2f(m[i] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          const float e = exp2f(x[i][j] - ref);
          sum += e;
          sm.s[a + 8 * i][b + 16 * j] = e;
        }
        l[i] = l[i] * shrink + sum;  // (this thread's keys; summed over the row at the end)
        m[i] = top;
#pragma unroll
        for (int j = 0; j < 4 * CJ; ++j) o[i][j] *= shrink;
      }
      __syncwarp();  // (a row of S is written and read by one half of a warp)
      bool fine = true;
      if (masked) {  // (0 x infinity: see below)
#pragma unroll 1
        for (int i = t; i < BN * DP / 4; i += PA_THREADS) {
          const float4 y = *reinterpret_cast<const float4*>(&sm.v[cur][i / (DP / 4)][i % (DP / 4) * 4]);
          fine = fine && fabsf(y.x) < CUDART_INF_F && fabsf(y.y) < CUDART_INF_F && fabsf(y.z) < CUDART_INF_F && fabsf(y.w) < CUDART_INF_F;
        }
        fine = __syncthreads_and(fine);
      }
      if (fine) pa_ffma_values<DP, RPT, BN, false>(sm.s, sm.v[cur], a, b, o);
      else pa_ffma_values<DP, RPT, BN, true>(sm.s, sm.v[cur], a, b, o);
      __syncwarp();
    }
    const bool whole = w.t0 == 0 && w.t1 == w.tiles;
    float* piece = pa_piece_of<RT, DP>(p, w);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = a + 8 * i;
      float sum = l[i];
#pragma unroll
      for (int k = 8; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      if (r >= w.rows) continue;
      if (whole) {
        T* out = reinterpret_cast<T*>(pa_out(p, w.s.start, w.head, w.row0 + r));
#pragma unroll
        for (int j = 0; j < 4 * CJ; ++j) {
          const int d = 4 * b + 64 * (j / 4) + j % 4;
          if (d < c.dim) pa_store(out + d, o[i][j] / sum);
        }
      } else {
#pragma unroll
        for (int j = 0; j < CJ; ++j)
          *reinterpret_cast<float4*>(piece + r * DP + 4 * b + 64 * j) = make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
        if (b == 0) {
          piece[RT * DP + r] = m[i];
          piece[RT * DP + RT + r] = sum;
        }
      }
    }
    cut.note(sm.share, w);
  }
}

// ---------------------------------------------------------------------------------------------- matrix-instruction forms
// Rows of whole 16-byte words. 16-bit types: rows of a tile in the M of mma m16n8k16, keys in its N (S = Q K^T) and then in
// its K (O += P V). Keys and values stay as they lie in the pages: cp.async brings rows of 2 DP bytes into a ring, 16-byte words
// at (word ^ row % 8), so that ldmatrix reads eight rows without bank conflicts; what a row of the table does not reach is zero.
// The softmax reference of a row is its running maximum, moved only when it grows by more than 2^8 (P then stays below 2^8, and
// a row of O is hardly ever rescaled); P is rounded to the cache's type as the operand of a matrix instruction has to be (half a step of
// bf16 or fp16: 2^-8, 2^-11 of a weight), its sum l is of the unrounded numbers in fp32. In fp16 all of P, l and O is taken 2^7 times, which
// the quotient does not see: P stays below 2^15, and what is too small for a normal number is off by 2^-32 of the largest weight at
// most (2^-25 otherwise: thousands of small weights beside a large one would be lost).
// fp32: every number is two of 11 bits, x = hi + lo with hi = x rounded to 11 bits, and a product the three of m16n8k8 (tf32) that
// lie above 2^-22 of it: hi hi + hi lo + lo hi. That keeps fp32's accuracy and takes a third of the instructions that fused
// multiply-adds of single lanes would. An infinity has no such halves, nor have the largest numbers: what sees one is NaN.
constexpr float PA_SLACK = 8.f;
template <typename T>
constexpr float PA_UP = std::is_same<T, __half>::value ? 7.f : 0.f;

__device__ __forceinline__ void pa_ldmatrix(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pa_ldmatrix_t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pa_finite_part(uint32_t x) {  // zero for a half that is an infinity or NaN
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return ((x & e) != e ? x & 0xffffu : 0u) | (((x >> 16) & e) != e ? x & 0xffff0000u : 0u);
}

// What one warp holds of 16 rows: thread (g = lane / 4, t = lane % 4) has rows g and g + 8.
template <typename T, int DP>
struct PaWarp {
  float o[DP / 8][4], m[2], l[2];
  uint32_t q[DP <= 128 ? DP / 16 : 1][4];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
  }

  // S = Q K^T for the NK keys at kt, P, and O += P V with the values at vt. q_at: Q in shared memory where it is too wide for
  // registers. hides (the same for the warp): row half h sees the keys of bits sees[h] only.
  template <int NK>
  __device__ __forceinline__ void step(uint32_t kt, uint32_t vt, float scale, uint32_t q_at, bool hides, const uint64_t (&sees)[2], float* spare) {
    const int lane = threadIdx.x & 31;
    float s[NK / 8][4];
#pragma unroll
    for (int n = 0; n < NK / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
    const int krow = (lane & 7) + ((lane >> 4) << 3), kword = (lane >> 3) & 1;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t a[4];
      if constexpr (DP <= 128) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = q[d][j];
      } else {
        const int r = lane & 15, w = 2 * d + (lane >> 4);
        pa_ldmatrix(q_at + r * (DP * 2) + ((w ^ (r & 7)) << 4), a);
      }
#pragma unroll
      for (int n = 0; n < NK / 16; ++n) {
        const int r = 16 * n + krow, w = 2 * d + kword;
        uint32_t b[4];
        pa_ldmatrix(kt + r * (DP * 2) + ((w ^ (r & 7)) << 4), b);
        pa_mma<T>(s[2 * n], a, b[0], b[1]);
        pa_mma<T>(s[2 * n + 1], a, b[2], b[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < NK / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] *= scale;
    bool fine = true;
    if (hides) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t mine = sees[h] >> (2 * (lane & 3));
#pragma unroll
        for (int n = 0; n < NK / 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (!((mine >> (8 * n + j)) & 1)) s[n][2 * h + j] = -CUDART_INF_F;
      }
      // A hidden row of V that is not finite would spoil every row (0 x infinity): such numbers are left out of the product
      // and added behind it, to the rows that see them.
#pragma unroll 1
      for (int i = lane; i < NK * DP / 8; i += 32) {
        uint4 x;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(vt + i * 16));
        fine = fine && pa_finite_part<T>(x.x) == x.x && pa_finite_part<T>(x.y) == x.y && pa_finite_part<T>(x.z) == x.z && pa_finite_part<T>(x.w) == x.w;
      }
      fine = __all_sync(0xffffffffu, fine);
    }
    float shrink[2];
    bool moves = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = -CUDART_INF_F;
#pragma unroll
      for (int n = 0; n < NK / 8; ++n) top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool up = top > m[h] + PA_SLACK || (m[h] == -CUDART_INF_F && top > m[h]);
      shrink[h] = up ? pa_exp2(m[h] - top) : 1.f;
      if (up) m[h] = top;
      moves = moves || up;
    }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] *= shrink[j >> 1];
      l[0] *= shrink[0];
      l[1] *= shrink[1];
    }
    const float ref[2] = {m[0] == -CUDART_INF_F ? 0.f : m[0] - PA_UP<T>, m[1] == -CUDART_INF_F ? 0.f : m[1] - PA_UP<T>};
#pragma unroll
    for (int n = 0; n < NK / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = pa_exp2(s[n][j] - ref[j >> 1]);
        l[j >> 1] += s[n][j];
      }
    const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3), vword = lane >> 4;
#pragma unroll
    for (int n = 0; n < NK / 16; ++n) {
      const uint32_t a[4] = {pa_pack<T>(s[2 * n][0], s[2 * n][1]), pa_pack<T>(s[2 * n][2], s[2 * n][3]),
                             pa_pack<T>(s[2 * n + 1][0], s[2 * n + 1][1]), pa_pack<T>(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const int r = 16 * n + vrow, w = 2 * d + vword;
        uint32_t b[4];
        pa_ldmatrix_t(vt + r * (DP * 2) + ((w ^ (r & 7)) << 4), b);
        if (!fine) {
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = pa_finite_part<T>(b[j]);
        }
        pa_mma<T>(o[2 * d], a, b[0], b[1]);
        pa_mma<T>(o[2 * d + 1], a, b[2], b[3]);
      }
    }
    if (!fine) add_infinite<NK>(s, vt, spare);
  }

  // O += P V for the numbers of V that are not finite and weights that are not zero. spare: 16 x 8 floats of the warp's own.
  template <int NK>
  __device__ __forceinline__ void add_infinite(const float (&s)[NK / 8][4], uint32_t vt, float* spare) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll 1
    for (int n = 0; n < NK / 8; ++n) {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < NK / 8; ++i)
          if (i == n) x = s[i][j];
        spare[(g + 8 * (j >> 1)) * 8 + 2 * t + (j & 1)] = x;
      }
      __syncwarp();
#pragma unroll 1
      for (int kk = 0; kk < 8; ++kk) {
        const float w0 = spare[g * 8 + kk], w1 = spare[(g + 8) * 8 + kk];
        const int r = 8 * n + kk;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          uint32_t x;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(vt + r * (DP * 2) + ((d ^ (r & 7)) << 4) + 4 * t));
          const uint32_t odd = x ^ pa_finite_part<T>(x);
          if (odd == 0) continue;
          T lo, hi;  // (the half that is finite, if one is, counts as zero)
          const uint16_t bits_lo = static_cast<uint16_t>(odd), bits_hi = static_cast<uint16_t>(odd >> 16);
          memcpy(&lo, &bits_lo, 2);
          memcpy(&hi, &bits_hi, 2);
          const float y0 = pa_load(&lo), y1 = pa_load(&hi);
          if (w0 != 0.f) {
            o[d][0] = fmaf(w0, y0, o[d][0]);
            o[d][1] = fmaf(w0, y1, o[d][1]);
          }
          if (w1 != 0.f) {
            o[d][2] = fmaf(w1, y0, o[d][2]);
            o[d][3] = fmaf(w1, y1, o[d][3]);
          }
        }
      }
    }
  }

  // Q of rows row .. row + 15 of the part (zero past the ends).
  __device__ __forceinline__ void load_q(const PaParams& p, const PaPart& w, int row) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row + (lane >> 2) + 8 * h, d0 = 2 * (lane & 3);
      const uint32_t* at = reinterpret_cast<const uint32_t*>(pa_query(p, w, min(r, w.rows_all - 1)) + 2 * d0);
#pragma unroll
      for (int d = 0; d < (DP <= 128 ? DP / 16 : 1); ++d) {
        q[d][h] = r < w.rows_all && 16 * d + d0 < p.c.dim ? at[8 * d] : 0u;
        q[d][2 + h] = r < w.rows_all && 16 * d + 8 + d0 < p.c.dim ? at[8 * d + 4] : 0u;
      }
    }
  }
  // The same into shared memory, `rows` rows by all threads of the CTA.
  static __device__ __forceinline__ void stage_q(const PaParams& p, const PaPart& w, void* into, int rows) {
    uint4* to = static_cast<uint4*>(into);
    for (int i = threadIdx.x; i < rows * (DP / 8); i += blockDim.x) {
      const int r = i / (DP / 8), x = i % (DP / 8);
      const bool there = w.row0 + r < w.rows_all && 8 * x < p.c.dim;
      to[r * (DP / 8) + (x ^ (r & 7))] = there ? reinterpret_cast<const uint4*>(pa_query(p, w, w.row0 + r))[x] : make_uint4(0u, 0u, 0u, 0u);
    }
  }

  __device__ __forceinline__ void finish_sums() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

// The same in fp32, eight keys a step; rows of the ring are 16 bytes longer than they have to be, so that the words of a fragment lie
// in different banks.
__device__ __forceinline__ void pa_mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (the instruction takes the upper 19 bits of an operand: what it leaves of lo is below 2^-22 of x)
__device__ __forceinline__ void pa_halves(float x, uint32_t* hi, uint32_t* lo) {
  *hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  *lo = __float_as_uint(x - __uint_as_float(*hi));
}
// Whether x has two halves: an infinity or NaN has none, nor has a number so near the largest one that hi would be an infinity.
__device__ __forceinline__ bool pa_halved(float x) { return fabsf(x) < 0x1.ffep127f; }
__device__ __forceinline__ float pa_lds(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at));
  return x;
}

template <int DP>
struct PaWarp<float, DP> {
  static constexpr int ROW = DP * 4 + 16;  // bytes of a row in the ring
  float o[DP / 8][4], m[2], l[2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    m[0] = m[1] = -CUDART_INF_F;
    l[0] = l[1] = 0.f;
  }

  // Q of 16 rows in the order of the fragments: for each step of 8 dims four words hi of every lane, then four lo.
  static __device__ __forceinline__ void stage_q(const PaParams& p, const PaPart& w, void* into, int) {
    uint4* to = static_cast<uint4*>(into);
    for (int i = threadIdx.x; i < DP / 8 * 32; i += blockDim.x) {
      const int lane = i & 31, d = i / 32 * 8 + (lane & 3);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = w.row0 + (lane >> 2) + 8 * (j & 1), dd = d + 4 * (j >> 1);
        const bool there = r < w.rows_all && dd < p.c.dim;
        pa_halves(there ? reinterpret_cast<const float*>(pa_query(p, w, r))[dd] : 0.f, &hi[j], &lo[j]);
      }
      to[i / 32 * 64 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      to[i / 32 * 64 + 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }

  template <int NK>
  __device__ __forceinline__ void step(uint32_t kt, uint32_t vt, float scale, uint32_t q_at, bool hides, const uint64_t (&sees)[2], float* spare) {
    static_assert(NK == 8, "one fragment of keys");
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float s[4];
    {
      float whole[2][4], cross[2][4];  // (sums of even and odd steps: four chains of instructions)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) whole[i][j] = cross[i][j] = 0.f;
      const uint32_t at = kt + g * ROW + 4 * t;
#pragma unroll
      for (int d0 = 0; d0 < DP / 8; d0 += 4) {  // (four steps' words first: the products wait for none)
        uint32_t ah[4][4], al[4][4], bh[4][2], bl[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = d0 + i;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(ah[i][0]), "=r"(ah[i][1]), "=r"(ah[i][2]), "=r"(ah[i][3]) : "r"(q_at + (d * 64 + lane) * 16));
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(al[i][0]), "=r"(al[i][1]), "=r"(al[i][2]), "=r"(al[i][3]) : "r"(q_at + (d * 64 + 32 + lane) * 16));
          pa_halves(pa_lds(at + 32 * d), &bh[i][0], &bl[i][0]);
          pa_halves(pa_lds(at + 32 * d + 16), &bh[i][1], &bl[i][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pa_mma_tf32(cross[i & 1], ah[i], bl[i][0], bl[i][1]);
          pa_mma_tf32(whole[i & 1], ah[i], bh[i][0], bh[i][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) pa_mma_tf32(cross[i & 1], al[i], bh[i][0], bh[i][1]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = ((cross[0][j] + cross[1][j]) + (whole[0][j] + whole[1][j])) * scale;
    }
    bool fine = true;
    if (hides) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!((sees[j >> 1] >> (2 * t + (j & 1))) & 1)) s[j] = -CUDART_INF_F;
#pragma unroll 1
      for (int i = lane; i < NK * DP; i += 32) fine = fine && pa_halved(pa_lds(vt + i / DP * ROW + i % DP * 4));
      fine = __all_sync(0xffffffffu, fine);
    }
    float shrink[2];
    bool moves = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = fmaxf(s[2 * h], s[2 * h + 1]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool up = top > m[h] + PA_SLACK || (m[h] == -CUDART_INF_F && top > m[h]);
      shrink[h] = up ? pa_exp2(m[h] - top) : 1.f;
      if (up) m[h] = top;
      moves = moves || up;
    }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] *= shrink[j >> 1];
      l[0] *= shrink[0];
      l[1] *= shrink[1];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = pa_exp2(s[j] - (m[j >> 1] == -CUDART_INF_F ? 0.f : m[j >> 1]));
      l[j >> 1] += s[j];
    }
    // keys 2 t and 2 t + 1, which this thread has weights of, are places t and t + 4 of the product
    uint32_t ah[4], al[4];
    pa_halves(s[0], &ah[0], &al[0]);
    pa_halves(s[2], &ah[1], &al[1]);
    pa_halves(s[1], &ah[2], &al[2]);
    pa_halves(s[3], &ah[3], &al[3]);
    const uint32_t at = vt + 2 * t * ROW + 4 * g;
#pragma unroll
    for (int d0 = 0; d0 < DP / 8; d0 += 4) {
      uint32_t bh[4][2], bl[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y[2] = {pa_lds(at + 32 * (d0 + i)), pa_lds(at + ROW + 32 * (d0 + i))};
        if (!fine) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (!pa_halved(y[j])) y[j] = 0.f;
        }
        pa_halves(y[0], &bh[i][0], &bl[i][0]);
        pa_halves(y[1], &bh[i][1], &bl[i][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pa_mma_tf32(o[d0 + i], ah, bl[i][0], bl[i][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) pa_mma_tf32(o[d0 + i], al, bh[i][0], bh[i][1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) pa_mma_tf32(o[d0 + i], ah, bh[i][0], bh[i][1]);
    }
    if (!fine) {  // as add_infinite of the 16-bit form
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) spare[(g + 8 * (j >> 1)) * 8 + 2 * t + (j & 1)] = s[j];
      __syncwarp();
#pragma unroll 1
      for (int kk = 0; kk < 8; ++kk) {
        const float w0 = spare[g * 8 + kk], w1 = spare[(g + 8) * 8 + kk];
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float y = pa_lds(vt + kk * ROW + (8 * d + 2 * t + j) * 4);
            if (pa_halved(y)) continue;
            if (w0 != 0.f) o[d][j] = fmaf(w0, y, o[d][j]);
            if (w1 != 0.f) o[d][2 + j] = fmaf(w1, y, o[d][2 + j]);
          }
      }
    }
  }

  __device__ __forceinline__ void finish_sums() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

// Up to 16 rows: every warp has its own keys (16 of each tile; 8 in fp32), its own ring, and no barrier until the part ends, where the
// warps' sums are joined. What bounds it is the copy of keys and values, 512 bytes a key and head at dim 128: 32 tokens behind up to 16384
// keys take 223 us, 6.2 TB/s, in a burst of 60 calls from a graph, and 229 to 246 call by call (dim 256: 4.6 TB/s). In fp32 (1024 bytes) it
// is the chain of instructions of a step, 800 for eight keys: 4.5 TB/s.
template <typename T, int DP>
struct PaNarrow {
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr int RT = 16, WARPS = !F32 || DP == 256 ? 4 : DP == 128 ? 12 : 16, THREADS = 32 * WARPS, CTAS = F32 || DP == 256 ? 1 : 2;
  static constexpr int KEYS = F32 ? 8 : 16, BN = WARPS * KEYS;
  // (fp32: as many warps as the shared memory and the registers hold; a step is a chain of instructions that wait for one another, and
  // 12 warps with two slots are faster than 8 with three: one node behind up to 32000 keys, 4 slots: 227 -> 174 us)
  static constexpr int STAGES = F32 ? 2 : DP == 64 ? 6 : 3, ROW = F32 ? DP * 4 + 16 : DP * 2, SLOT = KEYS * ROW;
  static constexpr int Q = F32 ? DP / 8 * 32 * 2 : DP > 128 ? 16 * DP / 8 : 1;
  uint4 ring[WARPS][STAGES][2][SLOT / 16];
  uint4 q[Q];
  float spare[WARPS][16 * 8];
  float m[WARPS][16], l[WARPS][16];
  uint32_t seen[RT][PA_TREE / 32 + 1];
  int16_t up[PA_TREE];
  PaShare share;
  // Where word `w` of row `r` lies in a slot.
  static __device__ __forceinline__ uint32_t at(int r, int w) { return r * ROW + ((F32 ? w : w ^ (r & 7)) << 4); }
};

template <typename T, int DP>
__global__ void __launch_bounds__(PaNarrow<T, DP>::THREADS, PaNarrow<T, DP>::CTAS) paged_attn_narrow_kernel(const PaParams p) {
  using S = PaNarrow<T, DP>;
  constexpr int RT = S::RT, BN = S::BN, ST = S::STAGES, KEYS = S::KEYS, WORDS = DP * sizeof(T) / 16;
  extern __shared__ __align__(128) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  pg_begin();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c4 = lane & 3;
  const PgCache& c = p.c;
  pa_share<RT, RT, BN>(p, &sm.share);
  const PaCut cut(p, threadIdx.x == 0);
  PaAt at(sm.share);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(sm.ring[warp]));
  const int words = c.dim * static_cast<int>(sizeof(T)) / 16;
  PaPart w;
  while (pa_next<RT, RT, BN>(p, &at, &w)) {
    const uint32_t mine = KEYS * warp;
    // (a lane looks up the page of key lane % KEYS of a step, one step before the copies need it)
    const auto lookup = [&](uint32_t tile) { return tile < w.t1 ? pa_lookup(p, w, tile * BN + mine + lane % KEYS) : -1; };
    uint32_t into = 0;  // ring slot of the next copies
    const auto fetch = [&](uint32_t tile, int pg) {
      if (tile < w.t1) {
        const PaRow r = pa_row(p, w, tile * BN + mine + lane % KEYS, pg);
        const uint32_t kt = ring + into * (2 * S::SLOT);
        const unsigned long long kp = reinterpret_cast<unsigned long long>(r.k), vp = reinterpret_cast<unsigned long long>(r.v);
#pragma unroll
        for (int i = 0; i < KEYS * WORDS / 32; ++i) {
          const int row = (32 * i + lane) / WORDS, word = (32 * i + lane) % WORDS;
          const unsigned long long a = __shfl_sync(0xffffffffu, kp, row), b = __shfl_sync(0xffffffffu, vp, row);
          const bool there = a != 0 && word < words;
          const uint32_t to = kt + S::at(row, word);
          pa_copy16(to, there ? reinterpret_cast<const char*>(a) + word * 16 : c.k.p, there);
          pa_copy16(to + S::SLOT, there ? reinterpret_cast<const char*>(b) + word * 16 : c.v.p, there);
        }
      }
      into = into == ST - 1 ? 0 : into + 1;
      pa_copy_commit();
    };
    __syncthreads();  // (the part before is done with the shared memory)
    PaWarp<T, DP> x;
    uint32_t q_at = 0;
    int pg = lookup(w.t0), node[2];
    const int words_seen = (w.s.nodes + 31) / 32, node0 = static_cast<int>(p.by_group.of(w.row0));
    // The first ST - 1 tiles are fetched by the loop itself, before there is one to work on.
#pragma unroll 1
    for (uint32_t tile = w.t0, out = 0; tile < w.t1 + ST - 1; ++tile) {
      const int next = lookup(tile + 1);
      fetch(tile, pg);
      pg = next;
      if (tile == w.t0 + ST - 2) {  // (behind the first copies)
        x.clear();
        if constexpr (S::Q == 1) {
          x.load_q(p, w, w.row0);
        } else {
          q_at = static_cast<uint32_t>(__cvta_generic_to_shared(sm.q));
          x.stage_q(p, w, sm.q, RT);
          __syncthreads();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) node[h] = static_cast<int>(p.by_group.of(w.row0 + min(g + 8 * h, w.rows - 1)));
        if (p.parents && static_cast<uint64_t>(w.t1) * BN > static_cast<uint32_t>(w.s.len))
          pa_ancestors(p, w.s, node0, min(RT, w.s.nodes - node0), sm.seen, sm.up);
      }
      if (tile < w.t0 + ST - 1) continue;
      pa_copy_wait<ST - 1>();
      __syncwarp();
      const uint32_t kt = ring + out * (2 * S::SLOT);
      out = out == ST - 1 ? 0 : out + 1;
      const int n0 = static_cast<int>((tile - (ST - 1)) * BN + mine) - w.s.len;  // the node at the first key
      if (n0 < w.s.nodes) {
        bool hides = n0 + KEYS > 0;
        uint64_t sees[2] = {0, 0};
        if (hides) {
#pragma unroll
          for (int h = 0; h < 2; ++h) sees[h] = pa_sees(p.parents ? sm.seen[node[h] - node0] : nullptr, words_seen, node[h], n0);
          hides = pa_any_hidden<KEYS>(sees);
        }
        x.template step<KEYS>(kt, kt + S::SLOT, p.scale, q_at, hides, sees, sm.spare[warp]);
      }
      __syncwarp();  // (the next copies go into the slot that has just been read)
    }
    pa_copy_wait<0>();
    x.finish_sums();
    // the warps' sums: O of each in its own ring
    __syncwarp();
    float* mine_o = reinterpret_cast<float*>(sm.ring[warp]);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(mine_o + (g + 8 * h) * DP + 8 * d + 2 * c4) = make_float2(x.o[d][2 * h], x.o[d][2 * h + 1]);
    if (c4 == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sm.m[warp][g + 8 * h] = x.m[h];
        sm.l[warp][g + 8 * h] = x.l[h];
      }
    }
    __syncthreads();
    const bool whole = w.t0 == 0 && w.t1 == w.tiles;
    float* piece = pa_piece_of<RT, DP>(p, w);
#pragma unroll 1
    for (int i = t; i < w.rows * (DP / 4); i += S::THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float m = -CUDART_INF_F;
#pragma unroll
      for (int k = 0; k < S::WARPS; ++k) m = fmaxf(m, sm.m[k][r]);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < S::WARPS; ++k) {
        const float mk = sm.m[k][r], f = mk == -CUDART_INF_F ? 0.f : pa_exp2(mk - m);
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[k]) + r * DP + d);
        l = fmaf(f, sm.l[k][r], l);
        o.x = fmaf(f, y.x, o.x);
        o.y = fmaf(f, y.y, o.y);
        o.z = fmaf(f, y.z, o.z);
        o.w = fmaf(f, y.w, o.w);
      }
      if (whole) {
        const float f = 1.f / l;
        char* out = pa_out(p, w.s.start, w.head, w.row0 + r) + d * sizeof(T);
        if (d >= c.dim) continue;
        if constexpr (S::F32) *reinterpret_cast<float4*>(out) = make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
        else *reinterpret_cast<uint2*>(out) = make_uint2(pa_pack<T>(o.x * f, o.y * f), pa_pack<T>(o.z * f, o.w * f));
      } else {
        *reinterpret_cast<float4*>(piece + r * DP + d) = o;
        if (d == 0) {
          piece[RT * DP + r] = m;
          piece[RT * DP + RT + r] = l;
        }
      }
    }
    cut.note(sm.share, w);
  }
}

// More than 16 rows of 136 to 256 dims (two streams as below would take 768 columns of tensor memory, which has 512): a warp for 16 of up
// to 128 rows (warps without rows only copy), all over the same tiles of keys. Bound by chains of instructions that wait for one another,
// two warps a scheduler (all that the registers hold): 256 rows of dim 256 behind 16000 keys, eight slots of eight heads, 1.44 ms, 187
// TFLOP/s (with four warps 2.66; mma.sync alone would take 0.5).
template <typename T>
struct PaWide {
  static constexpr int DP = 256, WARPS = 8, THREADS = 32 * WARPS, RT = 16 * WARPS, BN = 32, STAGES = 3, SLOT = BN * DP * 2;
  uint4 ring[STAGES][2][SLOT / 16];
  uint4 q[RT * DP * 2 / 16];
  const char* row[2][2][BN];  // (where the next tile's rows lie)
  float spare[WARPS][16 * 8];
  uint32_t seen[RT][PA_TREE / 32 + 1];
  int16_t up[PA_TREE];
  PaShare share;
};

template <typename T>
__global__ void __launch_bounds__(PaWide<T>::THREADS, 1) paged_attn_wide_kernel(const PaParams p) {
  using S = PaWide<T>;
  constexpr int DP = S::DP, RT = S::RT, BN = S::BN, ST = S::STAGES, WORDS = DP / 8, PER = S::THREADS / WORDS;
  static_assert(ST == 3, "two tiles on their way, one worked on");
  extern __shared__ __align__(128) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  pg_begin();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c4 = lane & 3;
  const PgCache& c = p.c;
  pa_share<RT, RT, BN>(p, &sm.share);
  const PaCut cut(p, threadIdx.x == 0);
  PaAt at(sm.share);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(sm.ring));
  const int word = t % WORDS, words = c.dim / 8;
  PaPart w;
  while (pa_next<RT, RT, BN>(p, &at, &w)) {
    const int words_seen = (w.s.nodes + 31) / 32;
    const int node0 = static_cast<int>(p.by_group.of(w.row0)), node1 = static_cast<int>(p.by_group.of(w.row0 + w.rows - 1));
    // Thread t < BN finds where row t of a tile lies, one tile before the copies of it, with the page that it looked up one tile
    // earlier still.
    int pg = t < BN ? pa_lookup(p, w, w.t0 * BN + t) : -1;
    const auto find = [&](uint32_t tile) {
      if (t < BN && tile < w.t1) {
        const PaRow r = pa_row(p, w, tile * BN + t, pg);
        sm.row[tile & 1][0][t] = r.k;
        sm.row[tile & 1][1][t] = r.v;
        if (tile + 1 < w.t1) pg = pa_lookup(p, w, (tile + 1) * BN + t);
      }
    };
    uint32_t into = 0;
    const auto fetch = [&](uint32_t tile) {
      if (tile < w.t1) {
        const uint32_t kt = ring + into * (2 * S::SLOT);
#pragma unroll
        for (int i = 0; i < BN / PER; ++i) {
          const int row = i * PER + t / WORDS;
          const char *a = sm.row[tile & 1][0][row], *b = sm.row[tile & 1][1][row];
          const bool there = a != nullptr && word < words;
          const uint32_t to = kt + row * (DP * 2) + ((word ^ (row & 7)) << 4);
          pa_copy16(to, there ? a + word * 16 : c.k.p, there);
          pa_copy16(to + S::SLOT, there ? b + word * 16 : c.v.p, there);
        }
      }
      into = into == ST - 1 ? 0 : into + 1;
      pa_copy_commit();
    };
    PaWarp<T, DP> x;
    uint32_t q_at = 0;
    int node[2];
    __syncthreads();  // (the part before is done with the shared memory)
    find(w.t0);
    // In round i tile i is fetched, the rows of tile i + 1 are found, and tile i - 2 is worked on.
#pragma unroll 1
    for (uint32_t tile = w.t0, out = 0; tile < w.t1 + ST - 1; ++tile) {
      pa_copy_wait<ST - 2>();
      __syncthreads();  // tile - 2 is there, tile - 3 has been read, and where the rows of `tile` lie has been written
      fetch(tile);
      find(tile + 1);
      if (tile == w.t0) {
        const int wrow = w.row0 + 16 * warp;
        x.clear();
        q_at = static_cast<uint32_t>(__cvta_generic_to_shared(sm.q)) + warp * 16 * (DP * 2);
        x.stage_q(p, w, sm.q, RT);
#pragma unroll
        for (int h = 0; h < 2; ++h) node[h] = static_cast<int>(p.by_group.of(min(wrow + g + 8 * h, w.rows_all - 1)));
        if (p.parents && static_cast<uint64_t>(w.t1) * BN > static_cast<uint32_t>(w.s.len)) pa_ancestors(p, w.s, node0, node1 - node0 + 1, sm.seen, sm.up);
      }
      if (tile < w.t0 + ST - 1) continue;
      const uint32_t kt = ring + out * (2 * S::SLOT);
      out = out == ST - 1 ? 0 : out + 1;
      const int n0 = static_cast<int>((tile - (ST - 1)) * BN) - w.s.len;
      if (16 * warp < w.rows) {
        bool hides = n0 + BN > 0;
        uint64_t sees[2] = {0, 0};
        if (hides) {
#pragma unroll
          for (int h = 0; h < 2; ++h) sees[h] = pa_sees(p.parents ? sm.seen[min(node[h], node1) - node0] : nullptr, words_seen, node[h], n0);
          hides = pa_any_hidden<BN>(sees);
        }
        x.template step<BN>(kt, kt + S::SLOT, p.scale, q_at, hides, sees, sm.spare[warp]);
      }
    }
    pa_copy_wait<0>();
    x.finish_sums();
    const bool whole = w.t0 == 0 && w.t1 == w.tiles;
    float* piece = pa_piece_of<RT, DP>(p, w);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * warp + g + 8 * h;
      if (r >= w.rows) continue;
      if (whole) {
        char* out = pa_out(p, w.s.start, w.head, w.row0 + r);
        const float f = 1.f / x.l[h];
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          if (8 * d < c.dim) *reinterpret_cast<uint32_t*>(out + 16 * d + 4 * c4) = pa_pack<T>(x.o[d][2 * h] * f, x.o[d][2 * h + 1] * f);
      } else {
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) *reinterpret_cast<float2*>(piece + r * DP + 8 * d + 2 * c4) = make_float2(x.o[d][2 * h], x.o[d][2 * h + 1]);
        if (c4 == 0) {
          piece[RT * DP + r] = x.m[h];
          piece[RT * DP + RT + r] = x.l[h];
        }
      }
    }
    cut.note(sm.share, w);
  }
}

// More than 16 rows: tcgen05. Two streams of blocks of 128 rows by 128 keys, whose scores S and sums O live in tensor memory: the two
// halves of up to 256 rows over the same keys or, where a part has no more than 128 rows, the even and the odd key tiles over the
// same rows, joined at its end. Keys and values come in tiles of 128 into shared memory, two of each: a tile of keys is free when its
// scores are there, one of values when its sums are. Two warps copy: tiles in front of the nodes by TMA, `box` rows of a page and 64
// dims an instruction (a box outside the pool reads zeros); tiles with nodes, and pages whose size is no multiple of 8, by cp.async,
// 16-byte words in the same 128-byte swizzle. One warp issues S_t = Q K^T and O_t += P_t V, and four warps for each stream turn S into
// P, a thread a row, while the tensor core works on the other stream. P stays in tensor memory, over its own scores. What bounds it is
// the chain S -> P -> O of a block, which two streams do not cover: 128 nodes x 4 heads behind 16000 keys, eight slots, take 318 us, 845
// TFLOP/s (0.50 of the tensor peak), where the products alone would take 160 us and the exponentials (four results a clock and quarter
// SM) 113; half a tile of rows, 32 nodes x 4 heads, 117 us, 4.5 TB/s.
template <typename T, int DP>
struct PaTc {
  static constexpr int RT = 256, RW = 128, BN = 128, THREADS = 384, STAGES = DP == 64 ? 4 : 2, TILE = 128 * DP * 2;
  static constexpr int K = 2 * TILE, V = K + STAGES * TILE, REST = V + STAGES * TILE;  // offsets: Q, keys, values, the rest
  struct Rest {
    uint64_t q_full, q_free, k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES], s_full[2], p_full[2], o_ready[2], o_free[2], met;
    uint32_t tmem;
    int stop;  // a wait has run out
    int odd[8];  // number of the part, from 1, in which a tile that was looked through had values that are not finite (by the part's number)
    float m[2][2][128], l[2][2][128];  // of the two streams over the same rows; by turns
    int16_t up[8][PA_TREE];            // a slot's parents, for each softmax warp
    PaShare share;
  };
  // (of the parts behind the one whose results a warp writes, the other stream may have weighed one, and the values of STAGES tiles, one of a
  // part at least, may be here)
  static_assert(STAGES + 2 <= 8, "numbers of parts at hand");
  static constexpr int BYTES = REST + static_cast<int>(sizeof(Rest)) + 1024;
  // Where 16-byte word `w` of row `r` of a tile lies.
  static __device__ __forceinline__ uint32_t at(int r, int w) { return (w >> 3) * (128 * 128) + r * 128 + (((w & 7) ^ (r & 7)) << 4); }
};

__device__ __forceinline__ uint64_t pa_pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void pa_unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t pa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The keys among 128 that a node sees, the first of them node n0 (negative: in front of the nodes). up: the slot's parents (nullptr:
// a chain).
__device__ __forceinline__ void pa_sees128(const int16_t* up, int node, int n0, uint32_t (&bits)[4]) {
  const int upto = up ? -n0 : node + 1 - n0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = upto - 32 * i;
    bits[i] = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1 : 0u;
  }
  if (up)
    for (int j = node; j >= 0 && j >= n0; j = up[j]) {
      const int b = j - n0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b >> 5 == i) bits[i] |= 1u << (b & 31);
    }
}

// A CTA of this kernel runs through its code once for a short call, at the speed at which instructions come from the L2 (0.6 us for
// 128 bytes of straight-line code were measured): what several places need is one loop or one function that is not inlined.
__device__ __noinline__ bool pa_wait_long(uint64_t* bar, uint32_t parity, volatile int* stop) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop)) != 0;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || pa_wait_long(bar, parity, stop);
}
// Half of a tile has landed: the issuer may have it. look_at: the tile holds values that not every row sees; one that is not finite must
// not meet a weight of zero: it is taken out here, and goes in at the end.
template <typename T, int DP>
__device__ __noinline__ void pa_tell(uint64_t* bar, uint32_t look_at, int half, int* odd, uint32_t part) {
  constexpr int WORDS = DP / 8, PER = 32 / WORDS;
  const int lane = threadIdx.x & 31, word = lane % WORDS;
  if (look_at) {
    bool any = false;
#pragma unroll 1
    for (int i0 = 0; i0 < 64 / PER; i0 += 4) {
      uint32_t at[4], x[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at[i] = look_at + PaTc<T, DP>::at(64 * half + (i0 + i) * PER + lane / WORDS, word);
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[i][0]), "=r"(x[i][1]), "=r"(x[i][2]), "=r"(x[i][3]) : "r"(at[i]) : "memory");
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bool here = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t y = pa_finite_part<T>(x[i][k]);
          here = here || y != x[i][k];
          x[i][k] = y;
        }
        if (here) asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at[i]), "r"(x[i][0]), "r"(x[i][1]), "r"(x[i][2]), "r"(x[i][3]) : "memory");
        any = any || here;
      }
    }
    if (__any_sync(0xffffffffu, any) && lane == 0) atomicExch(odd + part % 8, static_cast<int>(part + 1));
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}
// All rows of a part see the positions in front of this one: pa_tell looks through the key tiles from the one that it lies in on.
__device__ __forceinline__ int64_t pa_open(const PaParams& p, const PaPart& w) {
  return w.s.len + (p.parents ? 0 : static_cast<int64_t>(p.by_group.of(w.row0)) + 1);
}
// What the values that pa_tell took out of the part's tiles add to columns d .. d + 15 of a node's row: those of the nodes that it sees and,
// where the first of the tiles begins in front of the nodes, of the sequence's last positions, which all rows see. Up the tree once
// for 16 columns: at most 1024 nodes, or a chain's nodes from its row tile on, and 127 positions. Some milliseconds for the deepest tree; a
// walk for each key and column is longer than a wait may be.
template <typename T, int BN>
__device__ __noinline__ void pa_odd_values(const PaParams& p, const PaPart& w, const int16_t* up, int node, int d, float* sum) {
  const uint32_t t0 = max(w.t0, static_cast<uint32_t>(pa_open(p, w) / BN));
  const int begin = static_cast<int>(static_cast<int64_t>(t0) * BN - w.s.len), end = static_cast<int>(static_cast<int64_t>(w.t1) * BN - w.s.len);
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
  for (int j = up ? node : min(node, end - 1); j >= begin; j = up && j >= 0 ? up[j] : j - 1) {  // (-1 follows a root: the sequence)
    if (j >= end) continue;
    const uint32_t at = static_cast<uint32_t>(w.s.len + j);
    const char* const v = pa_row(p, w, at, pa_lookup(p, w, at)).v;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!v || d + 8 * k >= p.c.dim) continue;
      const uint4 x = *reinterpret_cast<const uint4*>(v + 2 * (d + 8 * k));
      const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t bits = static_cast<uint16_t>(y[e >> 1] >> (16 * (e & 1)));
        T z;
        memcpy(&z, &bits, 2);
        const float f = pa_load(&z);
        if (!(fabsf(f) < CUDART_INF_F)) sum[8 * k + e] += f;
      }
    }
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(PaTc<T, DP>::THREADS, 1)
    paged_attn_tc_kernel(const __grid_constant__ PaParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using S = PaTc<T, DP>;
  constexpr int RT = S::RT, RW = S::RW, BN = S::BN, ST = S::STAGES, TILE = S::TILE, WORDS = DP / 8, PER = 32 / WORDS;
  extern __shared__ __align__(128) unsigned char raw[];
  unsigned char* const smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  typename S::Rest& sm = *reinterpret_cast<typename S::Rest*>(smem + S::REST);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const PgCache& c = p.c;
  if (threadIdx.x == 0) {
    mbar_init(&sm.q_full, 2);  // (an arrival of each copying warp)
    mbar_init(&sm.q_free, 1);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&sm.k_full[s], 2);
      mbar_init(&sm.v_full[s], 2);
      mbar_init(&sm.k_free[s], 1);
      mbar_init(&sm.v_free[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_full[t], 4);  // (of each softmax warp of the stream)
      mbar_init(&sm.o_ready[t], 1);
      mbar_init(&sm.o_free[t], 8);  // (of all softmax warps, or twice of the stream's own)
    }
    mbar_init(&sm.met, 8);
    sm.stop = 0;
    for (int i = 0; i < 8; ++i) sm.odd[i] = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  pg_begin();
  pa_share<RT, RW, BN>(p, &sm.share);
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  // columns of tensor memory: S0 / P0 at 0, S1 / P1 at 128, O0 at 256, O1 at 384
  volatile int* const stop = &sm.stop;
  PaAt at(sm.share);
  PaPart w;
  uint32_t n_part = 0;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------ the issuer of the matrix instructions (all lanes, one leads)
    const uint32_t lead = lane == 0 ? 1u : 0u, q0 = smem_u32(smem), k0 = q0 + S::K, v0 = q0 + S::V;
    constexpr uint32_t FORMAT = std::is_same<T, __half>::value ? 0u : 1u;
    const uint32_t idesc_s = umma_idesc(FORMAT, 0, 0, 128, 128) | (p.scale < 0.f ? 1u << 13 : 0u), idesc_o = umma_idesc(FORMAT, 0, 1, 128, DP);
    uint32_t n_k = 0, n_v = 0;                 // key and value tiles so far
    uint32_t p_odd = 0, o_odd = 0, o_any = 0;  // bit t: of stream t, whether the P tiles, the results are odd in number; any results
    const auto issue_s = [&](int t, uint32_t qa, uint32_t stage) {
      const uint32_t ka = k0 + stage * TILE;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t o = (k >> 2) * (128 * 128) + (k & 3) * 32;
        tc_mma_f16_lead(tmem + 128 * t, umma_smem_desc_sw128(qa + o, 16, 1024), umma_smem_desc_sw128(ka + o, 16, 1024), idesc_s, k != 0, lead);
      }
      tc_commit_lead(smem_u32(&sm.s_full[t]), lead);
    };
    const auto issue_o = [&](int t, uint32_t stage, bool more) {
      const uint32_t va = v0 + stage * TILE;
#pragma unroll
      for (int k = 0; k < BN / 16; ++k)
        tc_mma_f16_ts_lead(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, umma_smem_desc_sw128(va + k * 2048, 128 * 128, 1024), idesc_o, more || k != 0, lead);
      tc_commit_lead(smem_u32(&sm.o_ready[t]), lead);
    };
    // P_t is there, and O_t may be written
    const auto weights = [&](int t, bool first) {
      if (!pa_wait(&sm.p_full[t], (p_odd >> t) & 1, stop)) return false;
      if (first && ((o_any >> t) & 1) && !pa_wait(&sm.o_free[t], ((o_odd >> t) & 1) ^ 1, stop)) return false;
      p_odd ^= 1u << t;
      tc_fence_after();
      return true;
    };
    while (ok && pa_next<RT, RW, BN>(p, &at, &w)) {
      // Blocks in the order of the streams 0, 1, 0, 1, ...: two row tiles of a key tile, or one row tile of two key tiles. Behind O of
      // a block comes S of the stream's next one, which overwrites P. `last`: the block is the last one of its key tile.
      const bool pair = w.rows > 128;
      const int n = static_cast<int>(w.t1 - w.t0) << (pair ? 1 : 0);
      if (!(ok = pa_wait(&sm.q_full, n_part & 1, stop))) break;
      for (int i = -2; i < n; ++i) {
        const int t = i & 1;
        const bool first = !pair || t == 0, last = !pair || t == 1;
        if (i >= 0) {
          const uint32_t s = n_v % ST;
          if (first && !(ok = pa_wait(&sm.v_full[s], (n_v / ST) & 1, stop))) break;
          if (!(ok = weights(t, i < 2))) break;
          issue_o(t, s, i > 1);
          if (last) {
            tc_commit_lead(smem_u32(&sm.v_free[s]), lead);
            ++n_v;
          }
        }
        if (i + 2 < n) {
          const uint32_t s = n_k % ST;
          if (first && !(ok = pa_wait(&sm.k_full[s], (n_k / ST) & 1, stop))) break;
          tc_fence_after();
          issue_s(t, q0 + (pair ? t * TILE : 0), s);
          if (last) {
            tc_commit_lead(smem_u32(&sm.k_free[s]), lead);
            ++n_k;
          }
          if (i + 3 == n) tc_commit_lead(smem_u32(&sm.q_free), lead);
        }
      }
      const uint32_t wrote = n > 1 ? 3u : 1u;
      o_odd ^= wrote;
      o_any |= wrote;
      ++n_part;
    }
  } else if (warp == 2 || warp == 3) {
    // ------------------------------------------------------------ copies: half of the rows of a tile each
    const int half = warp - 2, words = c.dim / 8, word = lane % WORDS;
    const uint32_t q0 = smem_u32(smem), k0 = q0 + S::K, v0 = q0 + S::V;
    uint32_t n_k = 0, n_v = 0;
    const PaCut cut(p, warp == 2 && lane == 0);
    const uint32_t lead = lane == 0 ? 1u : 0u;
    // A group of copies is told to the issuer when the next one is on its way, or before a wait.
    uint64_t* told = nullptr;
    uint32_t look_at = 0;  // (values of a tile with nodes)
    const auto flush = [&]() {
      if (told) {
        pa_copy_wait<0>();
        pa_tell<T, DP>(told, look_at, half, sm.odd, n_part);
        told = nullptr;
      }
    };
    const int my_boxes = p.box == 128 ? 1 - half : p.box ? 64 / p.box : 0;  // (a box that is a whole tile is fetched by one warp)
    while (ok && pa_next<RT, RW, BN>(p, &at, &w)) {
      const int64_t open = pa_open(p, w);
      // tiles in front of `plain` hold no nodes; pages of a tile, a lane a box or a lane two rows
      const uint32_t plain = p.box ? min(static_cast<uint32_t>(w.s.len) / BN, w.t1) : 0;
      const auto lookup = [&](uint32_t tile, int (&pg)[2]) {
        const bool boxes = tile < plain;
        const uint32_t x = tile * BN + 64 * half + lane * (boxes ? p.box : 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) pg[i] = tile < w.t1 && (!boxes || (i == 0 && lane < my_boxes)) ? pa_lookup(p, w, x + 32 * i) : -1;
      };
      const int n = w.t1 - w.t0, q_tiles = w.rows > 128 ? 2 : 1;
      int pages[2], pages_before[2] = {-1, -1}, pages_next[2] = {-1, -1};  // of key tile i, of the one before, of the next
      lookup(w.t0, pages);
      if (n_part > 0 && !(ok = pa_wait(&sm.q_free, (n_part - 1) & 1, stop))) break;
      // Q, then in round i keys of tile i and values of tile i - 1
#pragma unroll 1
      for (int z = -q_tiles; z < 2 * n + 2; ++z) {
        const bool v = z >= 0 && (z & 1);
        const int i = z >> 1, mine = v ? i - 1 : i;
        const uint32_t tile = w.t0 + mine;
        uint64_t* full = nullptr;
        uint32_t to, look = 0;
        unsigned long long from[2];
        if (z < 0) {
          const int qt = z + q_tiles;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = w.row0 + 128 * qt + 64 * half + 32 * x + lane;
            from[x] = row < w.rows_all ? reinterpret_cast<unsigned long long>(pa_query(p, w, row)) : 0;
          }
          to = q0 + qt * TILE;
          if (z == -1) full = &sm.q_full;
        } else {
          if (mine < 0 || mine >= n) {
            if (v) {
              pages_before[0] = pages[0], pages_before[1] = pages[1];
              pages[0] = pages_next[0], pages[1] = pages_next[1];
            }
            continue;
          }
          const uint32_t m = v ? n_v : n_k, s = m % ST;
          uint64_t* const free = v ? &sm.v_free[s] : &sm.k_free[s];
          full = v ? &sm.v_full[s] : &sm.k_full[s];
          to = (v ? v0 : k0) + s * TILE;
          const int pg[2] = {v ? pages_before[0] : pages[0], v ? pages_before[1] : pages[1]};
          if (!v) lookup(tile + 1, pages_next);
          if (!__all_sync(0xffffffffu, mbar_try_wait(free, ((m / ST) & 1) ^ 1))) {
            flush();
            if (!(ok = pa_wait(free, ((m / ST) & 1) ^ 1, stop))) break;
          }
          (v ? n_v : n_k) = m + 1;
          if (v) {
            pages_before[0] = pages[0], pages_before[1] = pages[1];
            pages[0] = pages_next[0], pages[1] = pages_next[1];
          }
          if (tile < plain) {
            const CUtensorMap* const map = v ? &map_v : &map_k;
            mbar_expect_tx_lead(smem_u32(full), static_cast<uint32_t>(my_boxes * p.box) * (DP / 64) * 128, lead);
            int mine_page = c.pages;  // (a page outside the pool reads zeros)
            if (lane < my_boxes && (mine_page = pa_checked(p, pg[0])) < 0) mine_page = c.pages;
            for (int x = 0; x < my_boxes; ++x) {
              const int row = 64 * half + x * p.box, page = __shfl_sync(0xffffffffu, mine_page, x);
#pragma unroll
              for (int d = 0; d < DP / 64; ++d)
                tma_load_4d_lead(to + d * (128 * 128) + row * 128, map, smem_u32(full), 64 * d, pg_row_of(c, tile * BN + row), w.head,
                                 page, lead);
            }
            flush();
            continue;
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const PaRow r = pa_row(p, w, tile * BN + 64 * half + 32 * x + lane, pg[x]);
            from[x] = reinterpret_cast<unsigned long long>(v ? r.v : r.k);
          }
          if (v && static_cast<int64_t>(tile + 1) * BN > open) look = to;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll 4
          for (int x = 0; x < 32 / PER; ++x) {
            const int r = x * PER + lane / WORDS;
            const unsigned long long a = __shfl_sync(0xffffffffu, from[h], r);
            const bool there = a != 0 && word < words;
            pa_copy16(to + S::at(64 * half + 32 * h + r, word), there ? reinterpret_cast<const char*>(a) + word * 16 : c.k.p, there);
          }
        if (!full) continue;  // (the second half of Q goes along)
        pa_copy_commit();
        if (told) {
          pa_copy_wait<1>();
          pa_tell<T, DP>(told, look_at, half, sm.odd, n_part);
        }
        told = full;
        look_at = look;
      }
      if (!ok) break;
      flush();
      cut.note(sm.share, w);
      ++n_part;
    }
    pa_copy_wait<0>();
    if (!ok) {  // copies in flight have to land before the CTA ends (again with a limit)
      const long long t0 = clock64();
      for (uint32_t i = n_k > ST ? n_k - ST : 0; i < n_k; ++i)
        while (!mbar_test_wait(&sm.k_full[i % ST], (i / ST) & 1) && clock64() - t0 < 20000000ll) {
        }
      for (uint32_t i = n_v > ST ? n_v - ST : 0; i < n_v; ++i)
        while (!mbar_test_wait(&sm.v_full[i % ST], (i / ST) & 1) && clock64() - t0 < 20000000ll) {
        }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax and results: stream t, a thread a row
    const int t = (warp - 4) >> 2, in_tile = (warp & 3) * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + 128 * t + lane_sel, to = tmem + 256 + 128 * t + lane_sel;
    const float scale = fabsf(p.scale);  // (a negative one: the instructions negate Q)
    uint32_t n_s = 0, n_other = 0, n_met = 0;  // score tiles of this stream and of the other one, parts with both streams over one row tile
    int16_t* const mine = sm.up[warp - 4];
    const int16_t* const up = p.parents ? mine : nullptr;
    while (ok && pa_next<RT, RW, BN>(p, &at, &w)) {
      const uint32_t all = w.t1 - w.t0;
      const bool split = w.rows <= 128;
      const int n = split ? (all - t + 1) / 2 : all;  // key tiles of this stream
      const bool nodes_here = static_cast<int64_t>(w.t1) * BN > w.s.len;
      if (p.parents && nodes_here) {
        __syncwarp();
        for (int i = lane; i < w.s.nodes; i += 32) {
          int a = p.parents[w.s.start + i];
          if (a < -1 || a >= i) {
            atomicOr(c.status, YTC_PAGES_INVALID);
            a = -1;
          }
          mine[i] = static_cast<int16_t>(a);
        }
        __syncwarp();
      }
      const int r = split ? in_tile : 128 * t + in_tile;
      const int node = static_cast<int>(p.by_group.of(w.row0 + min(r, w.rows - 1)));
      const bool idle = r - lane >= w.rows;  // no row of the warp is one: nobody reads its P
      float m = -CUDART_INF_F, l = 0.f;
      for (int j = 0; j < n; ++j, ++n_s) {
        if (!(ok = pa_wait(&sm.s_full[t], n_s & 1, stop))) break;
        if (idle) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[t]);
          continue;
        }
        tc_fence_after();
        const int n0 = static_cast<int>((w.t0 + (split ? 2 * j + t : j)) * BN) - w.s.len;
        bool masked = n0 + BN > 0;
        uint32_t bits[4];
        if (masked) {
          pa_sees128(up, node, n0, bits);
          masked = __any_sync(0xffffffffu, (bits[0] & bits[1] & bits[2] & bits[3]) != 0xffffffffu);
        }
        __syncwarp();
        if (masked) {  // what is hidden is -infinity from here on
#pragma unroll 1
          for (int k = 0; k < BN; k += 16) {
            const uint32_t b = (k < 64 ? k < 32 ? bits[0] : bits[1] : k < 96 ? bits[2] : bits[3]) >> (k & 16);
            uint32_t x[16];
            tmem_ld_32x32b_x16(ts + k, x);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = (b >> e) & 1 ? x[e] : __float_as_uint(-CUDART_INF_F);
            tmem_st_32x32b_x16(ts + k, x);
          }
          tmem_st_wait();
        }
        float top = -CUDART_INF_F;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t x[64];
          tmem_ld_32x32b_x64(ts + 64 * h, x);
          tmem_ld_wait();
          float a[4] = {top, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int e = 0; e < 64; e += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = pa_max3(a[k], __uint_as_float(x[e + 2 * k]), __uint_as_float(x[e + 2 * k + 1]));
          top = pa_max3(fmaxf(a[0], a[1]), a[2], a[3]);
        }
        top *= scale;
        if (j == 0) {
          m = top;
        } else {
          const bool moves = top > m + PA_SLACK || (m == -CUDART_INF_F && top > m);
          if (__any_sync(0xffffffffu, moves)) {  // O *= 2^(m - top): the product before has to be there
            if (!(ok = pa_wait(&sm.o_ready[t], (n_s - 1) & 1, stop))) break;
            tc_fence_after();
            const float shrink = moves ? pa_exp2(m - top) : 1.f;
#pragma unroll 1
            for (int d = 0; d < DP; d += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(to + d, x);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * shrink);
              tmem_st_32x32b_x16(to + d, x);
            }
            l *= shrink;
            if (moves) m = top;
          }
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m - PA_UP<T>;
        const uint64_t s2 = pa_pair(scale, scale), r2 = pa_pair(-ref, -ref);
        float l0 = 0.f, l1 = 0.f;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t x[64], pk[32];
          tmem_ld_32x32b_x64(ts + 64 * h, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            float a, b;
            pa_unpair(pa_fma2(pa_pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), s2, r2), a, b);
            a = pa_exp2(a);
            b = pa_exp2(b);
            l0 += a;
            l1 += b;
            pk[e >> 1] = pa_pack<T>(a, b);
          }
          // (P of the first half lies over scores that have been read: columns 0 .. 31)
          tmem_st_32x32b_x32(ts + 32 * h, pk);
        }
        l += l0 + l1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[t]);
      }
      if (!ok) break;
      // The sums: of this stream's own rows or, half of the columns each, of both streams over the same rows.
      float weight[2] = {1.f, 0.f};
      int d0 = 0, d1 = DP;
      if (split) {
        const int turn = n_met & 1;
        sm.m[turn][t][in_tile] = m;
        sm.l[turn][t][in_tile] = l;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.met);
        if (!(ok = pa_wait(&sm.met, n_met & 1, stop))) break;
        ++n_met;
        const float m0 = sm.m[turn][0][in_tile], m1 = sm.m[turn][1][in_tile];
        m = fmaxf(m0, m1);
        weight[0] = m0 == -CUDART_INF_F ? 0.f : pa_exp2(m0 - m);
        weight[1] = m1 == -CUDART_INF_F ? 0.f : pa_exp2(m1 - m);
        l = weight[0] * sm.l[turn][0][in_tile] + weight[1] * sm.l[turn][1][in_tile];
        d0 = t * (DP / 2);
        d1 = d0 + DP / 2;
        const int n1 = static_cast<int>(all / 2), n2 = static_cast<int>(all) - n1;  // key tiles of stream 1, of stream 0
        n_other += t ? n2 : n1;
        if ((t ? n2 : n1) > 0 && !(ok = pa_wait(&sm.o_ready[1 - t], (n_other - 1) & 1, stop))) break;
      } else {
        n_other += all;
      }
      if (n > 0 && !(ok = pa_wait(&sm.o_ready[t], (n_s - 1) & 1, stop))) break;
      tc_fence_after();
      const bool whole = w.t0 == 0 && w.t1 == w.tiles, here = r < w.rows, both = split && all > 1;
      const bool odd = *reinterpret_cast<volatile int*>(&sm.odd[n_part % 8]) == static_cast<int>(n_part + 1);
      float* const piece = pa_piece_of<RT, DP>(p, w);
      char* const out = here ? pa_out(p, w.s.start, w.head, w.row0 + r) : nullptr;
      const float f = 1.f / l;
      const uint32_t o0 = split ? tmem + 256 + lane_sel : to;
      if (!idle) {
#pragma unroll 1
        for (int d = d0; d < d1; d += 16) {
          uint32_t x[16];
          __syncwarp();
          tmem_ld_32x32b_x16(o0 + d, x);
          tmem_ld_wait();
          if (both) {
            uint32_t y[16];
            tmem_ld_32x32b_x16(o0 + 128 + d, y);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(weight[0] * __uint_as_float(x[e]) + weight[1] * __uint_as_float(y[e]));
          }
          if (odd && here) {
            float more[16];
            pa_odd_values<T, BN>(p, w, up, node, d, more);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) + more[e]);
          }
          if (here && whole) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (d + 8 * k < c.dim) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = pa_pack<T>(__uint_as_float(x[8 * k + 2 * e]) * f, __uint_as_float(x[8 * k + 2 * e + 1]) * f);
                *reinterpret_cast<uint4*>(out + 2 * (d + 8 * k)) = make_uint4(y[0], y[1], y[2], y[3]);
              }
          } else if (here) {
#pragma unroll
            for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(piece + r * DP + d + 4 * k) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
          }
        }
        if (here && !whole && d0 == 0) {
          piece[RT * DP + r] = m;
          piece[RT * DP + RT + r] = l;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        // O of a stream without key tiles in the part has not been written, and nobody waits for it to be read
        mbar_arrive(&sm.o_free[split ? 0 : t]);
        if (!split || both) mbar_arrive(&sm.o_free[split ? 1 : t]);
      }
      ++n_part;
    }
  }
  if (!ok && lane == 0) {
    *stop = 1;
    if (p.timeout) atomicExch(p.timeout, YTC_TIMEOUT);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------------------------- joining, storing
// New rows go to their pages, in `words` pieces of type W a head: warp number `warp` of `warps` takes every so manieth row and head.
template <typename W>
__device__ __forceinline__ void pa_store_new(const PaParams& p, int64_t warp, int64_t warps) {
  const PgCache& c = p.c;
  const int lane = threadIdx.x & 31, words = p.words;
  const int64_t items = static_cast<int64_t>(p.rows) * c.heads;
  for (int64_t i = warp; i < items; i += warps) {
    const int row = static_cast<int>(i / c.heads), head = static_cast<int>(i - static_cast<int64_t>(row) * c.heads);
    int slot = 0;  // slots that end at or before the row
    for (int s0 = 0; s0 < c.slots; s0 += 32) slot += __popc(__ballot_sync(0xffffffffu, s0 + lane < c.slots && p.starts[s0 + lane + 1] <= row));
    if (slot >= c.slots) continue;
    bool bad = false;
    const PaSlot s = pa_slot(p, slot, &bad);
    const int n = row - s.start;
    if (n < 0 || n >= s.nodes) continue;
    const int64_t at = static_cast<int64_t>(s.len) + n;
    const int pg = pg_page_of(c, slot, at);
    if (pg < 0 || c.refs[pg] != 1) {
      if (lane == 0) atomicOr(c.status, pg < 0 ? YTC_PAGES_INVALID : YTC_PAGES_SHARED);
      continue;
    }
    const int r = pg_row_of(c, at);
    const W* ks = reinterpret_cast<const W*>(p.k.p + row * p.k.row + head * p.k.head);
    const W* vs = reinterpret_cast<const W*>(p.v.p + row * p.v.row + head * p.v.head);
    W* kd = reinterpret_cast<W*>(c.k.p + pg * c.k.page + head * c.k.head + r * c.k.row);
    W* vd = reinterpret_cast<W*>(c.v.p + pg * c.v.page + head * c.v.head + r * c.v.row);
    for (int x = lane; x < 2 * words; x += 32) (x < words ? kd[x] : vd[x - words]) = x < words ? ks[x] : vs[x - words];
  }
}

constexpr int PA_JOIN = 256;  // threads of a CTA that joins
// CTAs (x, 0 .. joiners - 1) take their part of the unit that goes on behind share x: a unit's rows are dealt to the CTAs of all its
// shares but the last, so that the more pieces there are, the more CTAs join them (one sequence of 60,000 positions, one key head, 64
// nodes of 8 heads, bf16: 54 us instead of 167 with the CTAs of the first share alone). A row is one warp's work where the pieces are few
// or the rows many; else its pieces are dealt to the warps of a CTA, whose sums are joined in the order of the warps. Three reads that
// depend on one another: about 3 us behind the attention. CTAs (x, joiners ..) store the call's new rows at the same time.
template <typename T, int DP>
__global__ void __launch_bounds__(PA_JOIN) paged_attn_join_kernel(const PaParams p, int rt, int joiners) {
  constexpr int WARPS = PA_JOIN / 32, C4 = DP / 4, PER = (C4 + 31) / 32;
  __shared__ float sums[WARPS][DP + 1];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  pg_begin();
  if (static_cast<int>(blockIdx.y) >= joiners) {
    const int64_t at = (static_cast<int64_t>(blockIdx.y - joiners) * gridDim.x + blockIdx.x) * WARPS + warp;
    const int64_t all = static_cast<int64_t>(gridDim.y - joiners) * gridDim.x * WARPS;
    if (p.wide) pa_store_new<uint4>(p, at, all);
    else pa_store_new<T>(p, at, all);
    return;
  }
  const int4 a = p.cuts[2 * blockIdx.x], shares = p.cuts[2 * blockIdx.x + 1];
  if (a.x == 0) return;
  const int first = shares.x, pieces = shares.y - shares.x + 1;
  const int64_t size = pa_piece(rt, DP);
  // (the unit is the last of its first share and the first of the others)
  const float* const at = p.work + 2 * static_cast<int64_t>(first) * size;
  // The sums of pieces begin, begin + step, ... of row r, relative to the row's m.
  const auto gather = [&](int r, float m, int begin, int step, float* l, float4 (&o)[PER]) {
    *l = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = begin; i < pieces; i += step) {
      const float* x = at + (2 * i + (i == 0)) * size;
      const float mi = x[rt * DP + r], w = mi == -CUDART_INF_F ? 0.f : pa_exp2(mi - m);
      *l = fmaf(w, x[rt * DP + rt + r], *l);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (lane + 32 * j < C4) {
          const float4 y = *reinterpret_cast<const float4*>(x + r * DP + 4 * (lane + 32 * j));
          o[j].x = fmaf(w, y.x, o[j].x);
          o[j].y = fmaf(w, y.y, o[j].y);
          o[j].z = fmaf(w, y.z, o[j].z);
          o[j].w = fmaf(w, y.w, o[j].w);
        }
    }
  };
  const auto most = [&](int r) {
    float m = -CUDART_INF_F;
    for (int i = lane; i < pieces; i += 32) m = fmaxf(m, at[(2 * i + (i == 0)) * size + rt * DP + r]);
#pragma unroll
    for (int w = 16; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
    return m;
  };
  const int ctas = (pieces - 1) * joiners, cta = (static_cast<int>(blockIdx.x) - first) * joiners + blockIdx.y;
  if (pieces <= 8 || a.x > 2 * ctas) {  // (256 rows in three pieces took 17 us with a CTA a row)
    for (int r = warp * ctas + cta; r < a.x; r += ctas * WARPS) {
      float l;
      float4 o[PER];
      gather(r, most(r), 0, 1, &l, o);
      T* out = reinterpret_cast<T*>(pa_out(p, a.w, a.z, a.y + r));
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int d = 4 * (lane + 32 * j);
        const float y[4] = {o[j].x, o[j].y, o[j].z, o[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < p.c.dim) pa_store(out + d + e, y[e] / l);
      }
    }
    return;
  }
  for (int r = cta; r < a.x; r += ctas) {
    float l;
    float4 o[PER];
    gather(r, most(r), warp, WARPS, &l, o);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (lane + 32 * j < C4) {
        float* d = &sums[warp][4 * (lane + 32 * j)];
        d[0] = o[j].x;
        d[1] = o[j].y;
        d[2] = o[j].z;
        d[3] = o[j].w;
      }
    if (lane == 0) sums[warp][DP] = l;
    __syncthreads();
    T* out = reinterpret_cast<T*>(pa_out(p, a.w, a.z, a.y + r));
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all += sums[w][DP];
    for (int d = t; d < p.c.dim; d += PA_JOIN) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) x += sums[w][d];
      pa_store(out + d, x / all);
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
// How a call is cut: padded dim, rows and keys of a tile, CTAs.
struct PaForm {
  int dp, rt, bn, ctas, threads, smem;
  const void* kernel;
  bool boxes;      // the kernel takes tensor maps of keys and values
  int joiners = 1;  // CTAs of a share that join: one for 32 rows
};
template <typename... A>
static const void* pa_fn(void (*kernel)(A...)) {
  return reinterpret_cast<const void*>(kernel);
}

constexpr size_t PA_SHARED = 227 * 1024;  // what a CTA may have
template <typename T, int DP, int RPT>
static PaForm pa_ffma() {
  using S = PaFfma<T, DP, RPT>;
  static_assert(sizeof(S) <= PA_SHARED, "shared memory");
  const int smem = static_cast<int>(sizeof(S));
  return PaForm{DP, S::RT, S::BN, sm_count() * (smem <= 112 * 1024 ? 2 : 1), PA_THREADS, smem, pa_fn(paged_attn_ffma_kernel<T, DP, RPT>), false};
}
template <typename T, int DP>
static PaForm pa_form(int rows, bool words) {
  using N = PaNarrow<T, DP>;
  static_assert(N::CTAS * (sizeof(N) + 1024) <= PA_SHARED + 1024, "shared memory");
  if constexpr (sizeof(T) == 2) {
    if (words && rows > N::RT) {
      if constexpr (DP <= 128) {
        using C = PaTc<T, DP>;
        static_assert(C::BYTES <= PA_SHARED, "shared memory");
        return PaForm{DP, C::RT, C::BN, sm_count(), C::THREADS, C::BYTES, pa_fn(paged_attn_tc_kernel<T, DP>), true};
      } else {
        using W = PaWide<T>;
        static_assert(sizeof(W) <= PA_SHARED, "shared memory");
        return PaForm{DP, W::RT, W::BN, sm_count(), W::THREADS, static_cast<int>(sizeof(W)), pa_fn(paged_attn_wide_kernel<T>), false};
      }
    }
  }
  if (words) return PaForm{DP, N::RT, N::BN, sm_count() * N::CTAS, N::THREADS, static_cast<int>(sizeof(N)), pa_fn(paged_attn_narrow_kernel<T, DP>), false};
  return rows <= 8 ? pa_ffma<T, DP, 1>() : pa_ffma<T, DP, 4>();
}
template <typename T>
static PaForm pa_form(int dim, int rows, bool words) {
  return dim <= 64 ? pa_form<T, 64>(rows, words) : dim <= 128 ? pa_form<T, 128>(rows, words) : pa_form<T, 256>(rows, words);
}
// The form of a call: `rows` rows over the cache's slots, tiles of as many rows as a slot with an even share of them has. The host knows no
// more than that. One slot's tree in a cache of many idle ones is taken for few rows a slot: 32 nodes x 4 heads behind 16000 keys, 8 key
// heads, bf16, take 35 us on tcgen05 (a cache of one slot) and 94 in the narrow form (of 64 slots); behind 50 keys 25 and 15. `words`: all rows
// are whole 16-byte words on their boundaries.
static PaForm pa_choose(const ytcuda_pages* c, int rows, int heads, bool words) {
  const int64_t share = (static_cast<int64_t>(rows) + c->slots - 1) / c->slots * (heads / c->kv_heads);
  const int r = static_cast<int>(share < 4096 ? share : 4096);
  PaForm f = c->dtype == YTC_F32    ? pa_form<float>(c->dim, r, words)
             : c->dtype == YTC_BF16 ? pa_form<__nv_bfloat16>(c->dim, r, words)
                                    : pa_form<__half>(c->dim, r, words);
  f.joiners = ((r < f.rt ? r : f.rt) + 31) / 32;
  return f;
}
static uint64_t pa_pieces(const PaForm& f) { return 4ull * 2 * static_cast<uint64_t>(f.ctas) * static_cast<uint64_t>(pa_piece(f.rt, f.dp)); }
static uint64_t pa_space(const PaForm& f) { return pa_pieces(f) + 2ull * sizeof(int4) * static_cast<uint64_t>(f.ctas); }

// Tensor maps of a layer's keys and values, [pages, heads, rows of a page, dims], for boxes of 64 dims and as many rows as divide a
// page and a tile; 0 where that is no multiple of 8 (a swizzle's rows) or the strides allow no map.
static int pa_boxes(const PgCache& c, int dtype, CUtensorMap* k, CUtensorMap* v) {
  int rows = 128;
  while (c.page % rows) rows /= 2;
  if (rows < 8) return 0;
  const CUtensorMapDataType type = dtype == YTC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t dims[4] = {static_cast<uint64_t>(c.dim), static_cast<uint64_t>(c.page), static_cast<uint64_t>(c.heads), static_cast<uint64_t>(c.pages)};
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  for (const PgPool* p : {&c.k, &c.v}) {
    const uint64_t strides[3] = {static_cast<uint64_t>(p->row), static_cast<uint64_t>(p->head), static_cast<uint64_t>(p->page)};
    for (const uint64_t s : strides)
      if (s == 0 || s >= (1ull << 40)) return 0;
    if (encode_tensor_map(p == &c.k ? k : v, type, 4, p->p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B) != YTC_OK) return 0;
  }
  return rows;
}

template <typename T>
static cudaError_t pa_join(const PaForm& f, const PaParams& p, cudaStream_t st) {
  // a warp for each new row and head, up to eight rows of CTAs
  const int64_t stored = p.fresh ? (static_cast<int64_t>(p.rows) * p.c.heads - 1) / (f.ctas * (PA_JOIN / 32)) + 1 : 0;
  const dim3 grid(f.ctas, f.joiners + static_cast<int>(stored < 8 ? stored : 8)), block(PA_JOIN);
  if (f.dp == 64) return pg_launch(paged_attn_join_kernel<T, 64>, grid, block, 0, st, p, f.rt, f.joiners);
  if (f.dp == 128) return pg_launch(paged_attn_join_kernel<T, 128>, grid, block, 0, st, p, f.rt, f.joiners);
  return pg_launch(paged_attn_join_kernel<T, 256>, grid, block, 0, st, p, f.rt, f.joiners);
}

}  // namespace ytk

using namespace ytk;

extern "C" {

uint64_t ytcuda_pages_attend_workspace(const ytcuda_pages* cache, int rows, int heads) {
  if (!cache || rows <= 0 || heads <= 0 || cache->kv_heads <= 0 || cache->slots <= 0 || cache->dim <= 0) return 0;
  const uint64_t a = pa_space(pa_choose(cache, rows, heads, false)), b = pa_space(pa_choose(cache, rows, heads, true));
  return a > b ? a : b;
}

int ytcuda_pages_attend(const ytcuda_pages* cache, int layer, const void* q, void* o, const void* k, const void* v,
                        const int64_t* strides, const int32_t* starts, const int32_t* parents, int rows, int heads, float scale,
                        void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* who = "ytcuda_pages_attend";
  PaParams p{};
  if (const int rc = pg_take(who, cache, &p.c)) return rc;
  YTC_REQUIRE(layer >= 0 && layer < p.c.layers, "%s: layer %d of %d", who, layer, p.c.layers);
  YTC_REQUIRE(rows >= 0 && heads >= 1 && heads % p.c.heads == 0, "%s: %d rows of %d heads over %d key heads", who, rows, heads, p.c.heads);
  YTC_REQUIRE(static_cast<int64_t>(rows) * heads < (1ll << 31), "%s: %d rows of %d heads are too many", who, rows, heads);
  if (p.c.dim > 256) {
    set_last_error("%s: dim %d (at most 256)", who, p.c.dim);
    return YTC_UNSUPPORTED;
  }
  YTC_REQUIRE((k != nullptr) == (v != nullptr), "%s: k and v come together", who);
  if (rows == 0 || p.c.slots == 0) return YTC_OK;
  YTC_REQUIRE(starts && strides, "%s: null starts or strides", who);
  YTC_REQUIRE(p.c.pages > 0, "%s: a pool without pages", who);
  const int size = dtype_size(cache->dtype);
  if (const int rc = pg_rows(who, "q", q, strides, size, &p.q)) return rc;
  if (const int rc = pg_rows(who, "o", o, strides + 2, size, &p.o)) return rc;
  if (k) {
    if (const int rc = pg_rows(who, "k", k, strides + 4, size, &p.k)) return rc;
    if (const int rc = pg_rows(who, "v", v, strides + 6, size, &p.v)) return rc;
  }
  // (the CTAs write rows of o while others still read q, k and v; slices of one tensor that have no element in common are fine)
  const auto box = [&](const PgRows& r, int n) { return PgBox{r.p, {rows, n, 1, 1}, {r.row, r.head, 0, 0}, p.c.dim}; };
  YTC_REQUIRE(!pg_meet(box(p.o, heads), box(p.q, heads), size) && !pg_meet(box(p.o, heads), box(p.k, p.c.heads), size) &&
                  !pg_meet(box(p.o, heads), box(p.v, p.c.heads), size),
              "%s: o shares memory with q, k or v", who);
  // (a row behind row 0, a head behind head 0 of the same row)
  const PgBox row0{p.o.p, {1, heads, 1, 1}, {0, p.o.head, 0, 0}, p.c.dim}, head0{p.o.p, {1, 1, 1, 1}, {0, 0, 0, 0}, p.c.dim};
  const PgBox rows_behind{p.o.p + p.o.row, {rows - 1, heads, 1, 1}, {p.o.row, p.o.head, 0, 0}, p.c.dim};
  const PgBox heads_behind{p.o.p + p.o.head, {heads - 1, 1, 1, 1}, {p.o.head, 0, 0, 0}, p.c.dim};
  YTC_REQUIRE(!pg_meet(row0, rows_behind, size) && !pg_meet(head0, heads_behind, size), "%s: rows or heads of o lie in one another", who);
  const bool words = pg_width(pg_bits(p.c.k) | pg_bits(p.c.v) | pg_bits(p.q) | pg_bits(p.o) | pg_bits(p.k) | pg_bits(p.v) |
                              static_cast<uint64_t>(p.c.dim * size)) == 16;
  const PaForm f = pa_choose(cache, rows, heads, words);
  YTC_REQUIRE(workspace && workspace_bytes >= pa_space(f) && reinterpret_cast<uint64_t>(workspace) % 16 == 0,
              "%s: a workspace of %llu bytes on a 16-byte boundary is needed", who, static_cast<unsigned long long>(pa_space(f)));
  p.groups = heads / p.c.heads;
  // the most costs that the slots can have: row tiles of all slots, each over a full row of the table and its own nodes
  const int64_t row_tiles = static_cast<int64_t>(rows) * p.groups / f.rt * 3 + 3ll * p.c.slots;
  const int64_t key_tiles = (static_cast<int64_t>(p.c.max_pages) * p.c.page + rows) / f.bn + 1;
  if (static_cast<double>(row_tiles) * static_cast<double>(key_tiles) * p.c.heads >= 2147483648.0) {
    set_last_error("%s: %d rows over tables of %lld positions are too much work for one call", who, rows,
                   static_cast<long long>(p.c.max_pages) * p.c.page);
    return YTC_UNSUPPORTED;
  }
  p.c.k.p += layer * p.c.k.layer;
  p.c.v.p += layer * p.c.v.layer;
  p.by_group = pg_div(static_cast<uint32_t>(p.groups));
  p.starts = starts;
  p.parents = parents;
  p.rows = rows;
  p.fresh = k != nullptr;
  p.wide = words;
  p.words = words ? p.c.dim * size / 16 : p.c.dim;
  p.scale = (scale != 0.f ? scale : 1.f / sqrtf(static_cast<float>(p.c.dim))) * PA_LOG2E;
  p.work = static_cast<float*>(workspace);
  p.cuts = reinterpret_cast<int4*>(static_cast<char*>(workspace) + pa_pieces(f));
  p.timeout = device_status_word();
  if (!p.timeout) {
    set_last_error("%s: no device status word", who);
    return YTC_CUDA_ERROR;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (const int rc = ensure_dynamic_smem(f.kernel, f.smem)) return rc;
  CUtensorMap map_k{}, map_v{};
  if (f.boxes) p.box = pa_boxes(p.c, cache->dtype, &map_k, &map_v);
  void* args[] = {&p, &map_k, &map_v};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(f.ctas);
  cfg.blockDim = dim3(f.threads);
  cfg.dynamicSmemBytes = f.smem;
  cfg.stream = st;
  cudaLaunchAttribute overlapped[1];  // (as pg_launch)
  overlapped[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlapped[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = overlapped;
  cfg.numAttrs = 1;
  YTC_CUDA(cudaLaunchKernelExC(&cfg, f.kernel, args));
  count_launch();
  YTC_CUDA(cache->dtype == YTC_F32 ? pa_join<float>(f, p, st) : cache->dtype == YTC_BF16 ? pa_join<__nv_bfloat16>(f, p, st) : pa_join<__half>(f, p, st));
  count_launch();
  return YTC_OK;
}

}  // extern "C"
