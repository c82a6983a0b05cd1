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

#include "pages.cuh"

namespace ytk {

constexpr int PA_THREADS = 128;
constexpr int PA_TREE = 1024;  // most nodes of a tree
constexpr float PA_LOG2E = 1.4426950408889634f;

struct PaParams {
  PgCache c;  // (the pools at the layer)
  PgRows q, k, v, o;
  const int32_t *starts, *parents;
  int rows, heads, groups;
  int fresh;  // k and v hold the new rows: they are read from there, and stored
  float scale;  // times log2(e)
  float* work;
};

// What a slot brings: its rows in the call, its nodes, its length.
struct PaSlot {
  int start, nodes, len;
};
__device__ __forceinline__ PaSlot pa_slot(const PaParams& p, int s, bool* bad) {
  PaSlot r{p.starts[s], p.starts[s + 1], p.c.lens[s]};
  const int end = r.nodes;
  r.nodes = end - r.start;
  const bool ok = r.start >= 0 && end >= r.start && end <= p.rows && r.len >= 0 && !(p.parents && r.nodes > PA_TREE) &&
                  r.len + static_cast<int64_t>(p.fresh ? 0 : r.nodes) <= static_cast<int64_t>(p.c.held[s]) * p.c.page &&
                  p.c.held[s] <= p.c.max_pages;
  if (!ok) {
    *bad = *bad || r.nodes != 0;
    r.nodes = 0;
  }
  return r;
}
__device__ __forceinline__ int pa_key_tiles(const PaSlot& s, int bn) { return static_cast<int>((static_cast<int64_t>(s.len) + s.nodes + bn - 1) / bn); }
__device__ __forceinline__ int pa_row_tiles(const PaParams& p, const PaSlot& s, int rt) {
  return static_cast<int>((static_cast<int64_t>(s.nodes) * p.groups + rt - 1) / rt);
}
__device__ __forceinline__ int64_t pa_work(const PaParams& p, const PaSlot& s, int rt, int bn) {
  return s.nodes ? static_cast<int64_t>(pa_key_tiles(s, bn)) * pa_row_tiles(p, s, rt) * p.c.heads : 0;
}

// All key tiles of the call, and the slot that tile total * part / parts falls into with the tiles in front of it. For one warp.
struct PaPlace {
  int64_t total, at, before;
  int slot;
};
__device__ __forceinline__ PaPlace pa_place(const PaParams& p, int rt, int bn, int64_t part, int64_t parts, bool* bad) {
  const int lane = threadIdx.x & 31;
  PaPlace r{0, 0, 0, p.c.slots};
  for (int s0 = 0; s0 < p.c.slots; s0 += 32) {
    int64_t w = s0 + lane < p.c.slots ? pa_work(p, pa_slot(p, s0 + lane, bad), rt, bn) : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    r.total += w;
  }
  r.at = r.total * part / parts;
  int64_t before = 0;
  for (int s0 = 0; s0 < p.c.slots; s0 += 32) {
    const int64_t w = s0 + lane < p.c.slots ? pa_work(p, pa_slot(p, s0 + lane, bad), rt, bn) : 0;
    int64_t x = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + x > r.at);
    if (hit) {
      const int l = __ffs(hit) - 1;
      r.slot = s0 + l;
      r.before = before + __shfl_sync(0xffffffffu, x - w, l);
      return r;
    }
    before += __shfl_sync(0xffffffffu, x, 31);
  }
  return r;
}

// Floats of the workspace that one CTA has: two pieces (its first and its last unit may be cut) of O [rt][dp], m [rt], l [rt].
__host__ __device__ __forceinline__ int64_t pa_piece(int rt, int dp) { return static_cast<int64_t>(rt) * (dp + 2); }

// Element loads and stores in the cache's type; 16-bit results round to nearest even.
__device__ __forceinline__ float pa_load(const float* p) { return *p; }
__device__ __forceinline__ float pa_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float pa_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void pa_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void pa_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void pa_store(__half* p, float v) { *p = __float2half_rn(v); }

// Ancestors of the nodes of a row tile: bit j of seen[i - first] says that node j is node i or one of its ancestors. `up` takes
// the slot's parents. All threads of the CTA; a parent that is none counts as -1.
__device__ __forceinline__ void pa_ancestors(const PaParams& p, const PaSlot& s, int first, int count, uint32_t (*seen)[PA_TREE / 32], int16_t* up) {
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

// ---------------------------------------------------------------------------------------------- FFMA form
// fp32, and 16-bit rows that no matrix instruction takes (dims that are not a multiple of 8, odd alignments). 8 x 16 threads:
// thread (a, b) holds rows a + 8 i (RPT of them) with keys b + 16 j of S and with columns 4 b + 64 j of O.
template <int DP>
constexpr int PA_BN_F = DP == 256 ? 32 : 64;

template <typename T, int DP, int RPT>
struct PaSmemF {
  static constexpr int RT = 8 * RPT, BN = PA_BN_F<DP>;
  float q[RT][DP + 4], k[BN][DP + 4], v[BN][DP], s[RT][BN + 4];
  const T *kp[BN], *vp[BN];
  T *ks[BN], *vs[BN];
  uint32_t seen[RT][PA_TREE / 32];
  int16_t up[PA_TREE];
  int64_t from, to, before;
  int slot;
};

// O += S V of one tile. HIDDEN: weights of zero take nothing along (a hidden position may hold an infinity or NaN).
template <int DP, int RPT, int BN, bool HIDDEN>
__device__ __forceinline__ void pa_ffma_values(const float (*s)[BN + 4], const float (*v)[DP], int a, int b, float (*o)[DP / 16]) {
#pragma unroll 2
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
  using S = PaSmemF<T, DP, RPT>;
  constexpr int RT = S::RT, BN = S::BN, KPT = BN / 16, CJ = DP / 64;
  extern __shared__ __align__(16) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  dependent_trigger();
  const int t = threadIdx.x, a = t >> 4, b = t & 15;
  const PgCache& c = p.c;
  if (t < 32) {
    bool bad = false;
    const PaPlace at = pa_place(p, RT, BN, blockIdx.x, gridDim.x, &bad);
    if (__any_sync(0xffffffffu, bad) && t == 0 && blockIdx.x == 0) atomicOr(c.status, YTC_PAGES_INVALID);
    if (t == 0) {
      sm.from = at.at;
      sm.to = at.total * (blockIdx.x + 1) / gridDim.x;
      sm.before = at.before;
      sm.slot = at.slot;
    }
  }
  __syncthreads();
  int64_t pos = sm.from;
  const int64_t end = sm.to;
  int slot = sm.slot;
  int64_t off = pos - sm.before;
  while (pos < end) {
    bool bad = false;
    const PaSlot s = pa_slot(p, slot, &bad);
    const int64_t work = pa_work(p, s, RT, BN);
    if (off >= work) {  // (slots without rows too)
      off -= work;
      ++slot;
      continue;
    }
    const int tiles = pa_key_tiles(s, BN), row_tiles = pa_row_tiles(p, s, RT);
    const int unit = static_cast<int>(off / tiles), t0 = static_cast<int>(off - static_cast<int64_t>(unit) * tiles);
    const int t1 = static_cast<int>(end - pos < tiles - t0 ? t0 + (end - pos) : tiles);
    const int head = unit / row_tiles, rtile = unit - head * row_tiles;
    const int row0 = rtile * RT, rows = min(RT, s.nodes * p.groups - row0);
    const int keys = s.len + s.nodes;
    const int node0 = row0 / p.groups;
    __syncthreads();
    for (int i = t; i < RT * DP; i += PA_THREADS) {
      const int r = i / DP, d = i % DP;
      float x = 0.f;
      if (r < rows && d < c.dim) {
        const int node = (row0 + r) / p.groups, g = (row0 + r) % p.groups;
        x = pa_load(reinterpret_cast<const T*>(p.q.p + (s.start + node) * p.q.row + (head * p.groups + g) * p.q.head) + d);
      }
      sm.q[r][d] = x * p.scale;
    }
    if (p.parents && t1 * static_cast<int64_t>(BN) > s.len) pa_ancestors(p, s, node0, min(RT, s.nodes - node0), sm.seen, sm.up);
    float m[RPT], l[RPT], o[RPT][4 * CJ];
    int node[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      m[i] = -CUDART_INF_F;
      l[i] = 0.f;
      node[i] = (row0 + min(a + 8 * i, rows - 1)) / p.groups;
#pragma unroll
      for (int j = 0; j < 4 * CJ; ++j) o[i][j] = 0.f;
    }
    for (int tile = t0; tile < t1; ++tile) {
      const int k0 = tile * BN;
      __syncthreads();
      if (t < BN) {  // where the tile's rows are, and where they go
        const int at = k0 + t, j = at - s.len;
        const T *kp = nullptr, *vp = nullptr;
        T *ks = nullptr, *vs = nullptr;
        if (at < keys) {
          const int pg = j < 0 || !p.fresh || rtile == 0 ? pg_page_of(c, slot, at) : -1;
          const int64_t row = at % c.page;
          char* kc = c.k.p + pg * c.k.page + head * c.k.head + row * c.k.row;
          char* vc = c.v.p + pg * c.v.page + head * c.v.head + row * c.v.row;
          if (j >= 0 && p.fresh) {
            kp = reinterpret_cast<const T*>(p.k.p + (s.start + j) * p.k.row + head * p.k.head);
            vp = reinterpret_cast<const T*>(p.v.p + (s.start + j) * p.v.row + head * p.v.head);
            if (rtile == 0) {
              if (pg >= 0 && c.refs[pg] == 1) {
                ks = reinterpret_cast<T*>(kc);
                vs = reinterpret_cast<T*>(vc);
              } else {
                atomicOr(c.status, pg < 0 ? YTC_PAGES_INVALID : YTC_PAGES_SHARED);
              }
            }
          } else if (pg >= 0) {
            kp = reinterpret_cast<const T*>(kc);
            vp = reinterpret_cast<const T*>(vc);
          } else {
            atomicOr(c.status, YTC_PAGES_INVALID);
          }
        }
        sm.kp[t] = kp;
        sm.vp[t] = vp;
        sm.ks[t] = ks;
        sm.vs[t] = vs;
      }
      __syncthreads();
      for (int i = t; i < BN * DP; i += PA_THREADS) {
        const int r = i / DP, d = i % DP;
        float x = 0.f, y = 0.f;
        if (d < c.dim && sm.kp[r]) {
          const T xk = sm.kp[r][d], xv = sm.vp[r][d];
          x = pa_load(&xk);
          y = pa_load(&xv);
          if (sm.ks[r]) {
            sm.ks[r][d] = xk;
            sm.vs[r][d] = xv;
          }
        }
        sm.k[r][d] = x;
        sm.v[r][d] = y;
      }
      __syncthreads();
      float x[RPT][KPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < KPT; ++j) x[i][j] = 0.f;
#pragma unroll 4
      for (int d = 0; d < DP; d += 4) {
        float4 kk[KPT];
#pragma unroll
        for (int j = 0; j < KPT; ++j) kk[j] = *reinterpret_cast<const float4*>(&sm.k[b + 16 * j][d]);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(&sm.q[a + 8 * i][d]);
#pragma unroll
          for (int j = 0; j < KPT; ++j)
            x[i][j] = fmaf(qq.x, kk[j].x, fmaf(qq.y, kk[j].y, fmaf(qq.z, kk[j].z, fmaf(qq.w, kk[j].w, x[i][j]))));
        }
      }
      const bool masked = k0 + BN > s.len;
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        float top = m[i];
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          if (masked) {
            const int n = k0 + b + 16 * j - s.len;
            bool seen = n < 0;
            if (!seen && n < s.nodes) seen = p.parents ? (sm.seen[node[i] - node0][n >> 5] >> (n & 31)) & 1 : n <= node[i];
            if (!seen) x[i][j] = -CUDART_INF_F;
          }
          top = fmaxf(top, x[i][j]);
        }
#pragma unroll
        for (int w = 8; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
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
      if (masked) pa_ffma_values<DP, RPT, BN, true>(sm.s, sm.v, a, b, o);
      else pa_ffma_values<DP, RPT, BN, false>(sm.s, sm.v, a, b, o);
    }
    const bool whole = t0 == 0 && t1 == tiles;
    float* piece = p.work + (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0)) * pa_piece(RT, DP);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = a + 8 * i;
      float sum = l[i];
#pragma unroll
      for (int w = 8; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      if (r >= rows) continue;
      if (whole) {
        const int g = (row0 + r) % p.groups;
        T* out = reinterpret_cast<T*>(p.o.p + (s.start + node[i]) * p.o.row + (head * p.groups + g) * p.o.head);
#pragma unroll
        for (int j = 0; j < 4 * CJ; ++j) {
          const int d = 4 * b + 64 * (j / 4) + j % 4;
          if (d < c.dim) pa_store(out + d, o[i][j] / sum);
        }
      } else {
#pragma unroll
        for (int j = 0; j < CJ; ++j) *reinterpret_cast<float4*>(piece + r * DP + 4 * b + 64 * j) = make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
        if (b == 0) {
          piece[RT * DP + r] = m[i];
          piece[RT * DP + RT + r] = sum;
        }
      }
    }
    pos += t1 - t0;
    off += t1 - t0;
  }
}

// ---------------------------------------------------------------------------------------------- joining
// CTA (x, y): the unit that cut number x + 1 runs through, if it is the first one inside it; rows y, y + gridDim.y, ...; the
// pieces are shared by the warps, and their sums by way of shared memory joined in the order of the warps.
template <typename T, int DP>
__global__ void __launch_bounds__(PA_THREADS) paged_attn_join_kernel(const PaParams p, int rt, int bn, int parts) {
  constexpr int WARPS = PA_THREADS / 32, C4 = DP / 4, PER = (C4 + 31) / 32;
  __shared__ int64_t shared_at[3];
  __shared__ int shared_slot;
  __shared__ float sums[WARPS][DP + 1];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, cut = blockIdx.x + 1;
  if (t < 32) {
    bool bad = false;
    const PaPlace at = pa_place(p, rt, bn, cut, parts, &bad);
    if (t == 0) {
      shared_at[0] = at.total;
      shared_at[1] = at.at;
      shared_at[2] = at.before;
      shared_slot = at.slot;
    }
  }
  __syncthreads();
  dependent_wait();
  const int64_t total = shared_at[0], at = shared_at[1];
  const int slot = shared_slot;
  if (slot >= p.c.slots) return;
  bool bad = false;
  const PaSlot s = pa_slot(p, slot, &bad);
  const int tiles = pa_key_tiles(s, bn), row_tiles = pa_row_tiles(p, s, rt);
  const int64_t off = at - shared_at[2];
  const int unit = static_cast<int>(off / tiles), inside = static_cast<int>(off - static_cast<int64_t>(unit) * tiles);
  if (inside == 0 || total * (cut - 1) / parts > at - inside) return;
  const int64_t stop = at - inside + tiles;
  int last = cut;  // the last share that has tiles of the unit
  while (last + 1 < parts && total * (last + 1) / parts < stop) ++last;
  const int head = unit / row_tiles, row0 = (unit - head * row_tiles) * rt, rows = min(rt, s.nodes * p.groups - row0);
  const int64_t size = pa_piece(rt, DP);
  const auto piece = [&](int i) { return p.work + (2 * static_cast<int64_t>(i) + (i == cut - 1)) * size; };
  const auto empty = [&](int i) { return total * i / parts == total * (i + 1) / parts; };
  for (int r = blockIdx.y; r < rows; r += gridDim.y) {
    float m = -CUDART_INF_F;
    for (int i = cut - 1 + lane; i <= last; i += 32)
      if (!empty(i)) m = fmaxf(m, piece(i)[rt * DP + r]);
#pragma unroll
    for (int w = 16; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
    float l = 0.f;
    float4 o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = cut - 1 + warp; i <= last; i += WARPS) {
      if (empty(i)) continue;
      const float* x = piece(i);
      const float mi = x[rt * DP + r], w = mi == -CUDART_INF_F ? 0.f : exp2f(mi - m);
      l = fmaf(w, x[rt * DP + rt + r], l);
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
    const int node = (row0 + r) / p.groups, g = (row0 + r) % p.groups;
    T* out = reinterpret_cast<T*>(p.o.p + (s.start + node) * p.o.row + (head * p.groups + g) * p.o.head);
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all += sums[w][DP];
    for (int d = t; d < p.c.dim; d += PA_THREADS) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) x += sums[w][d];
      pa_store(out + d, x / all);
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
// How a call is cut: rows of a tile, padded dim, keys of a tile, CTAs.
struct PaForm {
  int rpt, dp, bn, rt, ctas, smem;
  const void* kernel;
};

template <typename T, int DP, int RPT>
static void pa_ffma(PaForm* f) {
  f->dp = DP;
  f->rpt = RPT;
  f->rt = 8 * RPT;
  f->bn = PA_BN_F<DP>;
  f->smem = static_cast<int>(sizeof(PaSmemF<T, DP, RPT>));
  f->kernel = reinterpret_cast<const void*>(paged_attn_ffma_kernel<T, DP, RPT>);
  f->ctas = sm_count() * (f->smem <= 110 * 1024 ? 2 : 1);
}
template <typename T>
static PaForm pa_form(int dim, int rows) {
  PaForm f{};
  if (dim <= 64) rows <= 8 ? pa_ffma<T, 64, 1>(&f) : rows <= 16 ? pa_ffma<T, 64, 2>(&f) : pa_ffma<T, 64, 4>(&f);
  else if (dim <= 128) rows <= 8 ? pa_ffma<T, 128, 1>(&f) : rows <= 16 ? pa_ffma<T, 128, 2>(&f) : pa_ffma<T, 128, 4>(&f);
  else rows <= 8 ? pa_ffma<T, 256, 1>(&f) : rows <= 16 ? pa_ffma<T, 256, 2>(&f) : pa_ffma<T, 256, 4>(&f);
  return f;
}
// The form of a call: `rows` rows over `slots` slots. Tiles of as many rows as a slot with an even share of them has.
static PaForm pa_choose(const ytcuda_pages* c, int rows, int heads) {
  const int share = c->slots ? (rows + c->slots - 1) / c->slots : 1;
  const int64_t tile = static_cast<int64_t>(share) * (heads / c->kv_heads);
  const int r = static_cast<int>(tile < 4096 ? tile : 4096);
  return c->dtype == YTC_F32 ? pa_form<float>(c->dim, r) : c->dtype == YTC_BF16 ? pa_form<__nv_bfloat16>(c->dim, r) : pa_form<__half>(c->dim, r);
}

template <typename T>
static cudaError_t pa_join(const PaForm& f, const PaParams& p, cudaStream_t st) {
  const dim3 grid(f.ctas - 1, f.rt < 16 ? f.rt : 16), block(PA_THREADS);
  if (f.dp == 64) return pg_launch_behind(paged_attn_join_kernel<T, 64>, grid, block, 0, st, p, f.rt, f.bn, f.ctas);
  if (f.dp == 128) return pg_launch_behind(paged_attn_join_kernel<T, 128>, grid, block, 0, st, p, f.rt, f.bn, f.ctas);
  return pg_launch_behind(paged_attn_join_kernel<T, 256>, grid, block, 0, st, p, f.rt, f.bn, f.ctas);
}

}  // namespace ytk

using namespace ytk;

extern "C" {

uint64_t ytcuda_pages_attend_workspace(const ytcuda_pages* cache, int rows, int heads) {
  if (!cache || rows <= 0 || heads <= 0 || cache->kv_heads <= 0 || cache->slots <= 0 || cache->dim <= 0) return 0;
  const PaForm f = pa_choose(cache, rows, heads);
  return 4ull * 2 * static_cast<uint64_t>(f.ctas) * static_cast<uint64_t>(pa_piece(f.rt, f.dp));
}

int ytcuda_pages_attend(const ytcuda_pages* cache, int layer, const void* q, const int64_t* q_strides, const void* k,
                        const int64_t* k_strides, const void* v, const int64_t* v_strides, void* o, const int64_t* o_strides,
                        const int32_t* starts, const int32_t* parents, int rows, int heads, float scale, void* workspace,
                        uint64_t workspace_bytes, void* stream) {
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
  YTC_REQUIRE(starts != nullptr, "%s: null starts", who);
  YTC_REQUIRE(p.c.pages > 0, "%s: a pool without pages", who);
  YTC_REQUIRE(q != o, "%s: q and o are the same memory", who);
  const int size = dtype_size(cache->dtype);
  if (const int rc = pg_rows(who, "q", q, q_strides, size, &p.q)) return rc;
  if (const int rc = pg_rows(who, "o", o, o_strides, size, &p.o)) return rc;
  if (k) {
    if (const int rc = pg_rows(who, "k", k, k_strides, size, &p.k)) return rc;
    if (const int rc = pg_rows(who, "v", v, v_strides, size, &p.v)) return rc;
  }
  const PaForm f = pa_choose(cache, rows, heads);
  YTC_REQUIRE(workspace && workspace_bytes >= ytcuda_pages_attend_workspace(cache, rows, heads) && reinterpret_cast<uint64_t>(workspace) % 16 == 0,
              "%s: a workspace of %llu bytes on a 16-byte boundary is needed", who,
              static_cast<unsigned long long>(ytcuda_pages_attend_workspace(cache, rows, heads)));
  p.c.k.p += layer * p.c.k.layer;
  p.c.v.p += layer * p.c.v.layer;
  p.starts = starts;
  p.parents = parents;
  p.rows = rows;
  p.heads = heads;
  p.groups = heads / p.c.heads;
  p.fresh = k != nullptr;
  p.scale = (scale != 0.f ? scale : 1.f / sqrtf(static_cast<float>(p.c.dim))) * PA_LOG2E;
  p.work = static_cast<float*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (const int rc = ensure_dynamic_smem(f.kernel, f.smem)) return rc;
  void* args[] = {&p};
  YTC_CUDA(cudaLaunchKernel(f.kernel, dim3(f.ctas), dim3(PA_THREADS), args, f.smem, st));
  count_launch();
  YTC_CUDA(cache->dtype == YTC_F32 ? pa_join<float>(f, p, st) : cache->dtype == YTC_BF16 ? pa_join<__nv_bfloat16>(f, p, st) : pa_join<__half>(f, p, st));
  count_launch();
  return YTC_OK;
}

}  // extern "C"
