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

// ---------------------------------------------------------------------------------------------- matrix-instruction forms
// 16-bit types with dims of whole 16-byte words: rows of a tile in the M of mma m16n8k16, keys in its N (S = Q K^T) and then in
// its K (O += P V). Keys and values stay as they lie in the pages: cp.async brings rows of 2 DP bytes into a ring, 16-byte words
// at (word ^ row % 8), so that ldmatrix reads eight rows without bank conflicts; what a row of the table does not reach is zero.
// The softmax reference of a row is its running maximum, moved only when it grows by more than 2^8 (P then stays below 2^8, and
// a row of O is hardly ever rescaled); P is rounded to the cache's type as the operand of a matrix instruction has to be, its sum
// l is of the unrounded numbers in fp32.
constexpr float PA_SLACK = 8.f;

__device__ __forceinline__ void pa_copy16(uint32_t dst, const char* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pa_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pa_copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pa_ldmatrix(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pa_ldmatrix_t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ bool pa_finite2(uint32_t x) {  // both halves
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return (x & e) != e && ((x >> 16) & e) != e;
}

template <typename T>
__device__ __forceinline__ uint32_t pa_finite_part(uint32_t x) {  // zero for a half that is none
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return ((x & e) != e ? x & 0xffffu : 0u) | (((x >> 16) & e) != e ? x & 0xffff0000u : 0u);
}

// Where the row of position `at` of a slot and head lies; nullptr where there is none. `pg`: its page, looked up before (-1: none).
struct PaRow {
  const char *k, *v;
};
__device__ __forceinline__ int pa_lookup(const PaParams& p, int slot, const PaSlot& s, int64_t at) {
  return at < s.len + static_cast<int64_t>(p.fresh ? 0 : s.nodes) ? pg_page_of(p.c, slot, at) : -1;
}
__device__ __forceinline__ PaRow pa_row(const PaParams& p, const PaSlot& s, int head, int64_t at, int pg) {
  PaRow r{nullptr, nullptr};
  if (pg >= 0) {
    const int row = static_cast<int>(at % p.c.page);
    r.k = p.c.k.p + pg * p.c.k.page + head * p.c.k.head + row * p.c.k.row;
    r.v = p.c.v.p + pg * p.c.v.page + head * p.c.v.head + row * p.c.v.row;
  } else if (p.fresh && at >= s.len && at < s.len + static_cast<int64_t>(s.nodes)) {
    const int64_t row = s.start + (at - s.len);
    r.k = p.k.p + row * p.k.row + head * p.k.head;
    r.v = p.v.p + row * p.v.row + head * p.v.head;
  }
  return r;
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

  // S = Q K^T for NK keys from shared row `key0` on, P, and O += P V. kt, vt: a ring slot's keys and values; q_at: Q in shared
  // memory where it is too wide for registers. seen(row half, key of the step): for steps that hide something.
  template <int NK, bool HIDES, typename Seen>
  __device__ __forceinline__ void step(uint32_t kt, uint32_t vt, int key0, float scale, uint32_t q_at, Seen seen, float* spare) {
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
        const int r = key0 + 16 * n + krow, w = 2 * d + kword;
        uint32_t b[4];
        pa_ldmatrix(kt + r * (DP * 2) + ((w ^ (r & 7)) << 4), b);
        pa_mma<T>(s[2 * n], a, b[0], b[1]);
        pa_mma<T>(s[2 * n + 1], a, b[2], b[3]);
      }
    }
    float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
    for (int n = 0; n < NK / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] *= scale;
        if (HIDES && !seen(j >> 1, 8 * n + 2 * (lane & 3) + (j & 1))) s[n][j] = -CUDART_INF_F;
        top[j >> 1] = fmaxf(top[j >> 1], s[n][j]);
      }
    float shrink[2];
    bool moves = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      const bool up = top[h] > m[h] + PA_SLACK || (m[h] == -CUDART_INF_F && top[h] > m[h]);
      shrink[h] = up ? pa_exp2(m[h] - top[h]) : 1.f;
      if (up) m[h] = top[h];
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
    const float ref[2] = {m[0] == -CUDART_INF_F ? 0.f : m[0], m[1] == -CUDART_INF_F ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < NK / 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[n][j] = pa_exp2(s[n][j] - ref[j >> 1]);
        l[j >> 1] += s[n][j];
      }
    // A hidden row of V that is not finite would spoil every row (0 x infinity): such numbers are left out of the product and
    // added behind it, to the rows that see them.
    bool fine = true;
    if (HIDES) {
      for (int i = lane; i < NK * DP / 8; i += 32) {
        uint4 x;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(vt + key0 * (DP * 2) + i * 16));
        fine = fine && pa_finite2<T>(x.x) && pa_finite2<T>(x.y) && pa_finite2<T>(x.z) && pa_finite2<T>(x.w);
      }
      fine = __all_sync(0xffffffffu, fine);
    }
    const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3), vword = lane >> 4;
#pragma unroll
    for (int n = 0; n < NK / 16; ++n) {
      const uint32_t a[4] = {pa_pack<T>(s[2 * n][0], s[2 * n][1]), pa_pack<T>(s[2 * n][2], s[2 * n][3]),
                             pa_pack<T>(s[2 * n + 1][0], s[2 * n + 1][1]), pa_pack<T>(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const int r = key0 + 16 * n + vrow, w = 2 * d + vword;
        uint32_t b[4];
        pa_ldmatrix_t(vt + r * (DP * 2) + ((w ^ (r & 7)) << 4), b);
        if (HIDES && !fine) {
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = pa_finite_part<T>(b[j]);
        }
        pa_mma<T>(o[2 * d], a, b[0], b[1]);
        pa_mma<T>(o[2 * d + 1], a, b[2], b[3]);
      }
    }
    if (HIDES && !fine) add_infinite<NK>(s, vt, key0, spare);
  }

  // O += P V for the numbers of V that are not finite and weights that are not zero. spare: 16 x 8 floats of the warp's own.
  template <int NK>
  __device__ __forceinline__ void add_infinite(const float (&s)[NK / 8][4], uint32_t vt, int key0, float* spare) {
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
        const int r = key0 + 8 * n + kk;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          uint32_t x;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(vt + r * (DP * 2) + ((d ^ (r & 7)) << 4) + 4 * t));
          if (pa_finite2<T>(x)) continue;
          const uint32_t odd = x ^ pa_finite_part<T>(x);  // (the finite half is zero)
          T lo, hi;
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

  __device__ __forceinline__ void finish_sums() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }
};

// Two neighbouring elements of a query row as one word (zero past the ends).
__device__ __forceinline__ uint32_t pa_q2(const PaParams& p, const PaSlot& s, int head, int row, int rows_all, int d) {
  if (row >= rows_all || d >= p.c.dim) return 0u;
  const int node = row / p.groups, g = row - node * p.groups;
  return *reinterpret_cast<const uint32_t*>(p.q.p + (s.start + static_cast<int64_t>(node)) * p.q.row + (head * p.groups + g) * p.q.head + 2 * d);
}

// Rows of new keys and values that a tile holds in shared memory go to their pages. `first` .. `first + n`: positions, `row0`: the
// shared row of the first; for `nt` threads of which this is number t.
template <int DP>
__device__ __forceinline__ void pa_store_new(const PaParams& p, const PaSlot& s, int slot, int head, int64_t first, int n, uint32_t kt,
                                             uint32_t vt, int row0, int t, int nt) {
  const int words = p.c.dim / 8;
  for (int i = t; i < n * words; i += nt) {
    const int r = i / words, w = i - r * words;
    const int64_t at = first + r;
    if (at < s.len || at >= s.len + static_cast<int64_t>(s.nodes)) continue;
    const int pg = pg_page_of(p.c, slot, at);
    if (pg < 0 || p.c.refs[pg] != 1) {
      atomicOr(p.c.status, pg < 0 ? YTC_PAGES_INVALID : YTC_PAGES_SHARED);
      continue;
    }
    const int row = static_cast<int>(at % p.c.page);
    const uint32_t off = (row0 + r) * (DP * 2) + ((w ^ ((row0 + r) & 7)) << 4);
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(kt + off));
    *reinterpret_cast<uint4*>(p.c.k.p + pg * p.c.k.page + head * p.c.k.head + row * p.c.k.row + w * 16) = x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(vt + off));
    *reinterpret_cast<uint4*>(p.c.v.p + pg * p.c.v.page + head * p.c.v.head + row * p.c.v.row + w * 16) = x;
  }
}

// Up to 16 rows: every warp has its own keys (16 of each tile of 64), its own ring, and no barrier until the unit ends, where the
// four warps' sums are joined. What bounds it is the copy of keys and values: 512 bytes a key and head at dim 128.
template <typename T, int DP>
struct PaNarrow {
  static constexpr int RT = 16, BN = 64, WARPS = 4, STAGES = DP == 64 ? 6 : 3, SLOT = 16 * DP * 2;  // bytes of 16 keys
  uint4 ring[WARPS][STAGES][2][SLOT / 16];
  uint4 q[DP > 128 ? 16 * DP * 2 / 16 : 1];
  float spare[WARPS][16 * 8];
  float m[WARPS][16], l[WARPS][16];
  uint32_t seen[RT][PA_TREE / 32];
  int16_t up[PA_TREE];
  int64_t from, to, before;
  int slot;
};

template <typename T, int DP>
__global__ void __launch_bounds__(PA_THREADS, DP == 256 ? 1 : 2) paged_attn_narrow_kernel(const PaParams p) {
  using S = PaNarrow<T, DP>;
  constexpr int RT = S::RT, BN = S::BN, ST = S::STAGES, WORDS = DP / 8, PER = 32 / WORDS;  // rows of a copy instruction
  extern __shared__ __align__(128) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  dependent_trigger();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c4 = lane & 3;
  const PgCache& c = p.c;
  if (warp == 0) {
    bool bad = false;
    const PaPlace at = pa_place(p, RT, BN, blockIdx.x, gridDim.x, &bad);
    if (__any_sync(0xffffffffu, bad) && lane == 0 && blockIdx.x == 0) atomicOr(c.status, YTC_PAGES_INVALID);
    if (lane == 0) {
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
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(sm.ring[warp]));
  const int word = lane % WORDS, words = c.dim / 8;
  while (pos < end) {
    bool bad = false;
    const PaSlot s = pa_slot(p, slot, &bad);
    const int64_t work = pa_work(p, s, RT, BN);
    if (off >= work) {
      off -= work;
      ++slot;
      continue;
    }
    const int tiles = pa_key_tiles(s, BN), row_tiles = pa_row_tiles(p, s, RT);
    const int unit = static_cast<int>(off / tiles), t0 = static_cast<int>(off - static_cast<int64_t>(unit) * tiles);
    const int t1 = static_cast<int>(end - pos < tiles - t0 ? t0 + (end - pos) : tiles);
    const int head = unit / row_tiles, rtile = unit - head * row_tiles;
    const int row0 = rtile * RT, rows_all = s.nodes * p.groups, rows = min(RT, rows_all - row0);
    const int64_t mine = 16 * warp;
    // (a lane looks up the page of key lane % 16 of a step, one step before the copies need it)
    const auto lookup = [&](int tile) { return tile < t1 ? pa_lookup(p, slot, s, static_cast<int64_t>(tile) * BN + mine + (lane & 15)) : -1; };
    const auto fetch = [&](int tile, int pg) {
      if (tile < t1) {
        const PaRow r = pa_row(p, s, head, static_cast<int64_t>(tile) * BN + mine + (lane & 15), pg);
        const uint32_t kt = ring + (tile - t0) % ST * (2 * S::SLOT);
        const unsigned long long kp = reinterpret_cast<unsigned long long>(r.k), vp = reinterpret_cast<unsigned long long>(r.v);
#pragma unroll
        for (int i = 0; i < 16 / PER; ++i) {
          const int row = i * PER + lane / WORDS;
          const unsigned long long a = __shfl_sync(0xffffffffu, kp, row), b = __shfl_sync(0xffffffffu, vp, row);
          const bool there = a != 0 && word < words;
          const uint32_t to = kt + row * (DP * 2) + ((word ^ (row & 7)) << 4);
          pa_copy16(to, there ? reinterpret_cast<const char*>(a) + word * 16 : c.k.p, there);
          pa_copy16(to + S::SLOT, there ? reinterpret_cast<const char*>(b) + word * 16 : c.v.p, there);
        }
      }
      pa_copy_commit();
    };
    __syncthreads();  // (the unit before is done with the shared memory)
    int pg = lookup(t0);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      const int next = lookup(t0 + i + 1);
      fetch(t0 + i, pg);
      pg = next;
    }
    PaWarp<T, DP> w;
    w.clear();
    uint32_t q_at = 0;
    if constexpr (DP <= 128) {
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) w.q[d][j] = pa_q2(p, s, head, row0 + g + 8 * (j & 1), rows_all, 16 * d + 2 * c4 + 8 * (j >> 1));
    } else {
      q_at = static_cast<uint32_t>(__cvta_generic_to_shared(sm.q));
      for (int i = t; i < 16 * DP / 2; i += PA_THREADS) {
        const int r = i / (DP / 2), d = i % (DP / 2) * 2;
        reinterpret_cast<uint32_t*>(sm.q)[r * (DP / 2) + (((d / 8) ^ (r & 7)) * 4) + d % 8 / 2] = pa_q2(p, s, head, row0 + r, rows_all, d);
      }
      __syncthreads();
    }
    const int node0 = row0 / p.groups;
    const int node[2] = {(row0 + min(g, rows - 1)) / p.groups, (row0 + min(g + 8, rows - 1)) / p.groups};
    if (p.parents && t1 * static_cast<int64_t>(BN) > s.len) pa_ancestors(p, s, node0, min(RT, s.nodes - node0), sm.seen, sm.up);
    for (int tile = t0; tile < t1; ++tile) {
      const int next = lookup(tile + ST);
      fetch(tile + ST - 1, pg);  // (into the slot that the step before has read)
      pg = next;
      pa_copy_wait<ST - 1>();
      __syncwarp();
      const uint32_t kt = ring + (tile - t0) % ST * (2 * S::SLOT), vt = kt + S::SLOT;
      const int64_t first = static_cast<int64_t>(tile) * BN + mine;
      if (first + 16 <= s.len) {
        w.template step<16, false>(kt, vt, 0, p.scale, q_at, [](int, int) { return true; }, nullptr);
      } else if (first < s.len + static_cast<int64_t>(s.nodes)) {
        const int before = static_cast<int>(s.len - first);
        w.template step<16, true>(
            kt, vt, 0, p.scale, q_at,
            [&](int h, int key) {
              const int n = key - before;
              if (n < 0) return true;
              if (n >= s.nodes) return false;
              return p.parents ? ((sm.seen[node[h] - node0][n >> 5] >> (n & 31)) & 1) != 0 : n <= node[h];
            },
            sm.spare[warp]);
        if (p.fresh && rtile == 0) pa_store_new<DP>(p, s, slot, head, first, 16, kt, vt, 0, lane, 32);
      }
      __syncwarp();
    }
    pa_copy_wait<0>();
    w.finish_sums();
    // the warps' sums: O of each in its own ring
    __syncwarp();
    float* mine_o = reinterpret_cast<float*>(sm.ring[warp]);
#pragma unroll
    for (int d = 0; d < DP / 8; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(mine_o + (g + 8 * h) * DP + 8 * d + 2 * c4) = make_float2(w.o[d][2 * h], w.o[d][2 * h + 1]);
    if (c4 == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sm.m[warp][g + 8 * h] = w.m[h];
        sm.l[warp][g + 8 * h] = w.l[h];
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    float* piece = p.work + (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0)) * pa_piece(RT, DP);
    for (int i = t; i < rows * (DP / 4); i += PA_THREADS) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float m = -CUDART_INF_F;
#pragma unroll
      for (int k = 0; k < S::WARPS; ++k) m = fmaxf(m, sm.m[k][r]);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < S::WARPS; ++k) {
        const float mk = sm.m[k][r], f = mk == -CUDART_INF_F ? 0.f : pa_exp2(mk - m);
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm.ring[k]) + r * DP + d);
        l = fmaf(f, sm.l[k][r], l);
        o.x = fmaf(f, x.x, o.x);
        o.y = fmaf(f, x.y, o.y);
        o.z = fmaf(f, x.z, o.z);
        o.w = fmaf(f, x.w, o.w);
      }
      if (whole) {
        if (d >= c.dim) continue;
        const int nd = (row0 + r) / p.groups, gg = (row0 + r) % p.groups;
        const float f = 1.f / l;
        *reinterpret_cast<uint2*>(p.o.p + (s.start + static_cast<int64_t>(nd)) * p.o.row + (head * p.groups + gg) * p.o.head + 2 * d) =
            make_uint2(pa_pack<T>(o.x * f, o.y * f), pa_pack<T>(o.z * f, o.w * f));
      } else {
        *reinterpret_cast<float4*>(piece + r * DP + d) = o;
        if (d == 0) {
          piece[RT * DP + r] = m;
          piece[RT * DP + RT + r] = l;
        }
      }
    }
    pos += t1 - t0;
    off += t1 - t0;
  }
}

// Up to 64 rows of a tile: a warp for 16 of them (warps without rows only copy), all over the same tiles of 64 keys.
template <typename T, int DP>
struct PaWide {
  static constexpr int RT = 64, BN = 64, STAGES = 3, SLOT = BN * DP * 2;
  uint4 ring[STAGES][2][SLOT / 16];
  uint4 q[DP > 128 ? RT * DP * 2 / 16 : 1];
  const char* row[2][2][BN];  // (where the next tile's rows lie)
  float spare[4][16 * 8];
  uint32_t seen[RT][PA_TREE / 32];
  int16_t up[PA_TREE];
  int64_t from, to, before;
  int slot;
};

template <typename T, int DP>
__global__ void __launch_bounds__(PA_THREADS, DP == 256 ? 1 : 2) paged_attn_wide_kernel(const PaParams p) {
  using S = PaWide<T, DP>;
  constexpr int RT = S::RT, BN = S::BN, ST = S::STAGES, WORDS = DP / 8, PER = PA_THREADS / WORDS;
  extern __shared__ __align__(128) unsigned char raw[];
  S& sm = *reinterpret_cast<S*>(raw);
  dependent_trigger();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c4 = lane & 3;
  const PgCache& c = p.c;
  if (warp == 0) {
    bool bad = false;
    const PaPlace at = pa_place(p, RT, BN, blockIdx.x, gridDim.x, &bad);
    if (__any_sync(0xffffffffu, bad) && lane == 0 && blockIdx.x == 0) atomicOr(c.status, YTC_PAGES_INVALID);
    if (lane == 0) {
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
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(sm.ring));
  const int word = t % WORDS, words = c.dim / 8;
  while (pos < end) {
    bool bad = false;
    const PaSlot s = pa_slot(p, slot, &bad);
    const int64_t work = pa_work(p, s, RT, BN);
    if (off >= work) {
      off -= work;
      ++slot;
      continue;
    }
    const int tiles = pa_key_tiles(s, BN), row_tiles = pa_row_tiles(p, s, RT);
    const int unit = static_cast<int>(off / tiles), t0 = static_cast<int>(off - static_cast<int64_t>(unit) * tiles);
    const int t1 = static_cast<int>(end - pos < tiles - t0 ? t0 + (end - pos) : tiles);
    const int head = unit / row_tiles, rtile = unit - head * row_tiles;
    const int row0 = rtile * RT, rows_all = s.nodes * p.groups, rows = min(RT, rows_all - row0);
    const int node_last = (row0 + rows - 1) / p.groups;
    // Thread t < 64 finds row t of a tile, one tile before the copies of it.
    const auto find = [&](int tile) {
      if (t < BN && tile < t1) {
        const int64_t at = static_cast<int64_t>(tile) * BN + t;
        const PaRow r = pa_row(p, s, head, at, pa_lookup(p, slot, s, at));
        sm.row[tile & 1][0][t] = r.k;
        sm.row[tile & 1][1][t] = r.v;
      }
    };
    const auto fetch = [&](int tile) {
      if (tile < t1) {
        const uint32_t kt = ring + (tile - t0) % ST * (2 * S::SLOT);
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
      pa_copy_commit();
    };
    __syncthreads();
    find(t0);
    find(t0 + 1);
    __syncthreads();
    fetch(t0);
    fetch(t0 + 1);
    __syncthreads();
    find(t0 + 2);
    PaWarp<T, DP> w;
    w.clear();
    const int wrow = row0 + 16 * warp;
    uint32_t q_at = 0;
    if constexpr (DP <= 128) {
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) w.q[d][j] = pa_q2(p, s, head, wrow + g + 8 * (j & 1), rows_all, 16 * d + 2 * c4 + 8 * (j >> 1));
    } else {
      q_at = static_cast<uint32_t>(__cvta_generic_to_shared(sm.q)) + warp * 16 * (DP * 2);
      for (int i = t; i < RT * DP / 2; i += PA_THREADS) {
        const int r = i / (DP / 2), d = i % (DP / 2) * 2;
        reinterpret_cast<uint32_t*>(sm.q)[r * (DP / 2) + (((d / 8) ^ (r & 7)) * 4) + d % 8 / 2] = pa_q2(p, s, head, row0 + r, rows_all, d);
      }
    }
    const int node0 = row0 / p.groups;
    const int node[2] = {min(wrow + g, rows_all - 1) / p.groups, min(wrow + g + 8, rows_all - 1) / p.groups};
    if (p.parents && t1 * static_cast<int64_t>(BN) > s.len) pa_ancestors(p, s, node0, node_last - node0 + 1, sm.seen, sm.up);
    for (int tile = t0; tile < t1; ++tile) {
      pa_copy_wait<ST - 2>();
      __syncthreads();  // the tile is there, the one before has been read, and where the next rows lie has been written
      fetch(tile + ST - 1);
      const uint32_t kt = ring + (tile - t0) % ST * (2 * S::SLOT), vt = kt + S::SLOT;
      const int64_t first = static_cast<int64_t>(tile) * BN;
      if (16 * warp < rows) {
        if (first + BN <= s.len) {
          w.template step<BN, false>(kt, vt, 0, p.scale, q_at, [](int, int) { return true; }, nullptr);
        } else if (first <= s.len + static_cast<int64_t>(node_last)) {
          const int before = static_cast<int>(s.len - first);
          w.template step<BN, true>(
              kt, vt, 0, p.scale, q_at,
              [&](int h, int key) {
                const int n = key - before;
                if (n < 0) return true;
                if (n > node_last) return false;
                return p.parents ? ((sm.seen[node[h] - node0][n >> 5] >> (n & 31)) & 1) != 0 : n <= node[h];
              },
              sm.spare[warp]);
        }
      }
      if (p.fresh && rtile == 0 && first + BN > s.len) pa_store_new<DP>(p, s, slot, head, first, BN, kt, vt, 0, t, PA_THREADS);
      find(tile + ST);
    }
    pa_copy_wait<0>();
    w.finish_sums();
    const bool whole = t0 == 0 && t1 == tiles;
    float* piece = p.work + (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0)) * pa_piece(RT, DP);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 16 * warp + g + 8 * h;
      if (r >= rows) continue;
      if (whole) {
        char* out = p.o.p + (s.start + static_cast<int64_t>(node[h])) * p.o.row + (head * p.groups + (row0 + r) % p.groups) * p.o.head;
        const float f = 1.f / w.l[h];
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
          if (8 * d < c.dim) *reinterpret_cast<uint32_t*>(out + 16 * d + 4 * c4) = pa_pack<T>(w.o[d][2 * h] * f, w.o[d][2 * h + 1] * f);
      } else {
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) *reinterpret_cast<float2*>(piece + r * DP + 8 * d + 2 * c4) = make_float2(w.o[d][2 * h], w.o[d][2 * h + 1]);
        if (c4 == 0) {
          piece[RT * DP + r] = w.m[h];
          piece[RT * DP + RT + r] = w.l[h];
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
template <typename T, int DP>
static void pa_mma_form(PaForm* f, int rows) {
  f->dp = DP;
  f->ctas = sm_count() * (DP == 256 ? 1 : 2);
  if (rows <= 16) {
    f->rt = PaNarrow<T, DP>::RT;
    f->bn = PaNarrow<T, DP>::BN;
    f->smem = static_cast<int>(sizeof(PaNarrow<T, DP>));
    f->kernel = reinterpret_cast<const void*>(paged_attn_narrow_kernel<T, DP>);
  } else {
    f->rt = PaWide<T, DP>::RT;
    f->bn = PaWide<T, DP>::BN;
    f->smem = static_cast<int>(sizeof(PaWide<T, DP>));
    f->kernel = reinterpret_cast<const void*>(paged_attn_wide_kernel<T, DP>);
  }
}
template <typename T>
static PaForm pa_form(int dim, int rows, bool words) {
  PaForm f{};
  if constexpr (sizeof(T) == 2) {
    if (words) {
      dim <= 64 ? pa_mma_form<T, 64>(&f, rows) : dim <= 128 ? pa_mma_form<T, 128>(&f, rows) : pa_mma_form<T, 256>(&f, rows);
      return f;
    }
  }
  if (dim <= 64) rows <= 8 ? pa_ffma<T, 64, 1>(&f) : rows <= 16 ? pa_ffma<T, 64, 2>(&f) : pa_ffma<T, 64, 4>(&f);
  else if (dim <= 128) rows <= 8 ? pa_ffma<T, 128, 1>(&f) : rows <= 16 ? pa_ffma<T, 128, 2>(&f) : pa_ffma<T, 128, 4>(&f);
  else rows <= 8 ? pa_ffma<T, 256, 1>(&f) : rows <= 16 ? pa_ffma<T, 256, 2>(&f) : pa_ffma<T, 256, 4>(&f);
  return f;
}
// The form of a call: `rows` rows over `slots` slots. Tiles of as many rows as a slot with an even share of them has. `words`: all
// rows are whole 16-byte words on their boundaries.
static PaForm pa_choose(const ytcuda_pages* c, int rows, int heads, bool words) {
  const int share = c->slots ? (rows + c->slots - 1) / c->slots : 1;
  const int64_t tile = static_cast<int64_t>(share) * (heads / c->kv_heads);
  const int r = static_cast<int>(tile < 4096 ? tile : 4096);
  return c->dtype == YTC_F32    ? pa_form<float>(c->dim, r, words)
         : c->dtype == YTC_BF16 ? pa_form<__nv_bfloat16>(c->dim, r, words)
                                : pa_form<__half>(c->dim, r, words);
}
static uint64_t pa_space(const PaForm& f) { return 4ull * 2 * static_cast<uint64_t>(f.ctas) * static_cast<uint64_t>(pa_piece(f.rt, f.dp)); }

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
  const uint64_t a = pa_space(pa_choose(cache, rows, heads, false)), b = pa_space(pa_choose(cache, rows, heads, true));
  return a > b ? a : b;
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
  const bool words = pg_width(pg_bits(p.c.k) | pg_bits(p.c.v) | pg_bits(p.q) | pg_bits(p.o) | pg_bits(p.k) | pg_bits(p.v) |
                              static_cast<uint64_t>(p.c.dim * size)) == 16;
  const PaForm f = pa_choose(cache, rows, heads, words);
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
