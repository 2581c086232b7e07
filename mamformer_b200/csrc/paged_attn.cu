// Attention over the paged 8-bit cache (layout in paged.cuh), for few query rows per KV head: single
// tokens and short runs of tokens.  Reads every key and value byte once.
//
//   S = scale q . (s_k k),  P = 2^(S log2 e - m),  O = sum P s_v v / sum P,   causal, optional window;
//   differential: (O1 - lam O2) / (1 - lam + 1e-8)
//
// The work is the list of (sequence, KV head, row tile) items, each a run of 64-token tiles; the grid's
// CTAs take equal contiguous shares of that list, so one long sequence fills the GPU as well as many short
// ones.  An item that ends in another CTA than it began in leaves partial (m, l, O) in a workspace and a
// second small kernel joins them in order (results do not depend on timing).
//
// A CTA is 4 warps; warp w takes tokens 16 w .. 16 w + 15 of each tile through a ring of its own, filled
// with 16-byte cp.async, and never waits for the other warps inside an item.  A warp's 16 tokens are the M
// rows of mma.m16n8k16 (f16 operands, fp32 sums): S^T = K Q^T and O^T = V^T P^T with up to 8 query rows as
// N, so 8 rows (4 heads of a group x 2 maps) fill the instruction; 16 rows take two.  e4m3 is exact in f16,
// and the rows of q are scaled by a power of two to [1, 2) first, which f16 holds exactly down to 2^-14 of a
// row's largest value.  P is rounded to f16 (11 bits; 8 in bf16).  The order of the head's dims in the
// products is free as long as both sides agree: a lane takes 16 adjacent bytes of K (and of V), so a
// fragment is loaded with one 16-byte read and no shuffles.
#include "paged.cuh"

namespace mamf {
namespace pa {

using namespace paged;

constexpr int NW = 4, NT = NW * 32;
constexpr int TILE = 16 * NW;                  // tokens per tile
constexpr float LAZY = 8.f;                    // log2 by which a row may outgrow its reference maximum

__device__ int g_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

struct Params {
  Cache c;
  const void *q1, *q2;
  void* out;
  const float* lam;
  int64_t st1, sh1, st2, sh2;
  int H, rep, maps, window, ctas;
  float scale_log2;
  float* part;        // [ctas][2][rows][HD + 2]: O (not divided), m, l
  int4* joins;        // [ctas]: the item that ends in this CTA after it began in another one
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
// two e4m3 codes -> two f16 values (exact)
__device__ __forceinline__ uint32_t to_h2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values held as mma fragments
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One row tile of one KV head of one sequence.
struct Item {
  int b, g, rt;
  int t0, n, len;            // first packed token, new tokens, cached length
  int rows;                  // n * rep * maps
  int lo, hi, k0, nt;        // slots [lo, hi) that some row of the tile sees, first tile, tiles (at least 1)
};

template <int ROWS>
__device__ __forceinline__ void set_range(const Params& p, Item& it) {
  const int per = p.rep * p.maps, first = it.len - it.n;
  const int i0 = it.rt * ROWS / per, i1 = min(it.n - 1, (it.rt * ROWS + ROWS - 1) / per);
  it.hi = max(0, min(it.len, first + i1 + 1));
  it.lo = p.window > 0 ? max(0, first + i0 - p.window + 1) : 0;
  it.k0 = it.lo / TILE;
  it.nt = it.hi > it.lo ? (it.hi + TILE - 1) / TILE - it.k0 : 1;
}
template <int ROWS>
__device__ __forceinline__ bool set_sequence(const Params& p, Item& it, int b) {
  it.b = b;
  it.t0 = p.c.cu[b];
  it.n = p.c.cu[b + 1] - it.t0;
  it.len = p.c.lens[b];
  if (it.n <= 0 || it.t0 < 0 || it.t0 + it.n > p.c.T) return false;
  it.rows = it.n * p.rep * p.maps;
  it.g = it.rt = 0;
  set_range<ROWS>(p, it);
  return true;
}
template <int ROWS>
__device__ __forceinline__ void next_item(const Params& p, Item& it) {
  if ((it.rt + 1) * ROWS < it.rows) { ++it.rt; set_range<ROWS>(p, it); return; }
  if (it.g + 1 < p.c.G) { ++it.g; it.rt = 0; set_range<ROWS>(p, it); return; }
  int b = it.b + 1;
  while (b < p.c.B && !set_sequence<ROWS>(p, it, b)) ++b;
  it.b = b;
}
template <int ROWS>
__device__ __forceinline__ int64_t tiles_of(const Params& p, int b) {
  Item it;
  if (!set_sequence<ROWS>(p, it, b)) return 0;
  int64_t n = 0;
  for (it.rt = 0; it.rt * ROWS < it.rows; ++it.rt) {
    set_range<ROWS>(p, it);
    n += it.nt;
  }
  return n * p.c.G;
}

template <int HD, int NR> constexpr int stage_bytes() { return 2 * 16 * HD + 16; }
template <int HD, int NR> constexpr int merge_floats() { return NW * 8 * NR * (HD + 4) + 2 * NW * 8 * NR; }
constexpr int STAGES = 3;
template <int HD, int NR> constexpr int smem_bytes() { return NW * STAGES * stage_bytes<HD, NR>() + 4 * merge_floats<HD, NR>(); }

// byte offset of 16-byte chunk c of token row r in a 16-token slice, arranged so that the 8 lanes of each
// phase of a 16-byte read (K: rows 2x, chunks of 4 lanes; V: rows 0, 2, 4, 6, two chunks) hit all banks once
template <int HD> __device__ __forceinline__ int k_at(int r, int c) {
  if (HD == 128) return r * 128 + ((c ^ ((r & 1) << 2)) << 4);
  return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (2 * ((r >> 1) & 3))) << 4);
}
template <int HD> __device__ __forceinline__ int v_at(int r, int c) {
  if (HD == 128) return r * 128 + ((c ^ (((r >> 1) & 3) << 1)) << 4);
  return k_at<HD>(r, c);
}

template <typename T> __device__ __forceinline__ void q_row16(const T* q, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Vec16<T> v = ld16(q + 8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[8 * i + j] = to_f(v.v[j]);
  }
}

template <typename T, int HD, int NR>
__global__ void __launch_bounds__(NT) split_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NR;
  constexpr int KC = HD / 64;                    // 16-byte reads of a K row per lane
  constexpr int MT = HD / 16;                    // 16-dim tiles of O^T
  constexpr int SB = stage_bytes<HD, NR>();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t s_pre[NT / 32];
  __shared__ int64_t s_begin;
  __shared__ int s_b;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  const Cache& c = p.c;
  asm volatile("griddepcontrol.launch_dependents;");      // the join kernel waits for this grid's end by itself

  // ---- this CTA's share [first, last) of the list of tiles ----
  const int chunk = (c.B + NT - 1) / NT;
  int64_t mine = 0;
  for (int i = 0; i < chunk; ++i) {
    const int b = tid * chunk + i;
    if (b < c.B) mine += tiles_of<ROWS>(p, b);
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_pre[w] = incl;
  if (tid == 0) s_b = -1;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (i < w) before += s_pre[i];
    total += s_pre[i];
  }
  incl += before;
  const int64_t share = (total + p.ctas - 1) / p.ctas;
  const int64_t first = blockIdx.x * share, last = min(total, first + share);
  if (incl - mine <= first && first < incl) {      // one thread at most
    int64_t at = incl - mine;
    int b = tid * chunk;
    for (;; ++b) {
      const int64_t n = tiles_of<ROWS>(p, b);
      if (first < at + n) break;
      at += n;
    }
    s_b = b;
    s_begin = at;
  }
  __syncthreads();
  if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
  // rows past the last sequence
  {
    const int end = c.B > 0 ? max(0, c.cu[c.B]) : 0;
    const int64_t n = (int64_t)max(0, c.T - end) * p.H * HD;
    for (int64_t i = (int64_t)blockIdx.x * NT + tid; i < n; i += (int64_t)gridDim.x * NT)
      ((T*)p.out)[(int64_t)end * p.H * HD + i] = from_f<T>(0.f);
  }
  if (first >= last) return;

  Item it;                                          // of the tile being computed
  set_sequence<ROWS>(p, it, s_b);
  int64_t start = s_begin;                          // list position of the item's first tile
  while (first >= start + it.nt) { start += it.nt; next_item<ROWS>(p, it); }

  // ---- ring: the issue side runs STAGES - 1 tiles ahead ----
  const uint32_t ring = su32(smem) + w * STAGES * SB;
  Item is = it;
  int is_tile = (int)(first - start);
  int64_t issued = first;
  auto page_of = [&](const Item& x, int tile) {
    const int slot = (x.k0 + tile) * TILE + w * 16;
    if (slot >= x.hi || slot + 16 <= x.lo) return -2;              // nothing to see in this slice
    const int j = slot >> c.shift;
    const int pg = j < c.W ? c.table[(int64_t)x.b * c.W + j] : -1;
    return (pg < 0 || pg >= c.P) ? -1 : pg;
  };
  int pg_next = page_of(is, is_tile);
  uint32_t live_bits = 0;                                           // which ring slots hold a slice
  auto issue = [&](int stage) {
    live_bits &= ~(1u << stage);
    if (issued < last) {
      if (pg_next >= 0) {
        const int slot = (is.k0 + is_tile) * TILE + w * 16;
        const int64_t blk = (int64_t)pg_next * c.G + is.g;
        const int64_t off = (blk * c.page + (slot & (c.page - 1))) * HD;
        const uint32_t dst = ring + stage * SB;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          const int idx = i * 32 + lane, r = idx / (HD / 16), cc = idx % (HD / 16);
          cp16(dst + k_at<HD>(r, cc), c.k + off + idx * 16);
          cp16(dst + 16 * HD + v_at<HD>(r, cc), c.v + off + idx * 16);
        }
        if (lane < 2) cp4(dst + 32 * HD + lane * 4, (lane ? c.vs : c.ks) + blk);
        live_bits |= 1u << stage;
      } else if (pg_next == -1 && lane == 0) record(ERR_PAGE);
      if (++issued < last) {
        if (++is_tile == is.nt) { next_item<ROWS>(p, is); is_tile = 0; }
        pg_next = page_of(is, is_tile);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);

  // ---- state of the current item ----
  uint32_t qf[NR][KC * 4][2];
  float rs[NR][2];                        // score factor of rows 2 t4, 2 t4 + 1
  int lim[NR][2], low[NR][2];             // slots (low, lim] that the row sees
  float m[NR][2], l[NR][2], o[NR][MT][4];
  float vref = 0.f;
  auto load_rows = [&]() {
    const int per = p.rep * p.maps;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int r = it.rt * ROWS + nr * 8 + g8;
      float f[KC][16];
      float mx = 0.f;
      if (r < it.rows) {
        const int i = r / per, h = it.g * p.rep + (r % per) / p.maps, map = r % p.maps;
        const T* q = map ? (const T*)p.q2 + (int64_t)(it.t0 + i) * p.st2 + (int64_t)h * p.sh2
                         : (const T*)p.q1 + (int64_t)(it.t0 + i) * p.st1 + (int64_t)h * p.sh1;
#pragma unroll
        for (int cc = 0; cc < KC; ++cc) q_row16(q + cc * 64 + t4 * 16, f[cc]);
#pragma unroll
        for (int cc = 0; cc < KC; ++cc)
#pragma unroll
          for (int j = 0; j < 16; ++j) mx = fmaxf(mx, fabsf(f[cc][j]));
      } else {
#pragma unroll
        for (int cc = 0; cc < KC; ++cc)
#pragma unroll
          for (int j = 0; j < 16; ++j) f[cc][j] = 0.f;
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^e <= mx < 2^(e + 1); rows of zeros and rows with infinities stay as they are
      int e = (int)(__float_as_uint(mx) >> 23) - 127;
      if (e == -127 || e == 128) e = 0;
      e = max(-126, min(126, e));
      const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
      for (int cc = 0; cc < KC; ++cc)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qf[nr][cc * 4 + i][0] = pack_h2(f[cc][4 * i] * down, f[cc][4 * i + 1] * down);
          qf[nr][cc * 4 + i][1] = pack_h2(f[cc][4 * i + 2] * down, f[cc][4 * i + 3] * down);
        }
      const float mine_rs = p.scale_log2 * up;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        rs[nr][x] = __shfl_sync(0xffffffffu, mine_rs, (2 * t4 + x) * 4);
        const int rr = it.rt * ROWS + nr * 8 + 2 * t4 + x;
        // rows past the last one are rows of zeros that see everything: they ask for no mask and are not written
        lim[nr][x] = rr < it.rows ? min(it.len - 1, it.len - it.n + rr / per) : 0x7fffffff;
        low[nr][x] = rr < it.rows && p.window > 0 ? it.len - it.n + rr / per - p.window : -1;
        m[nr][x] = -INFINITY;
        l[nr][x] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[nr][j][x] = 0.f;
    }
    vref = 0.f;
  };

  auto compute = [&](int stage, int slot0) {
    const uint32_t kb = ring + stage * SB, vb = kb + 16 * HD;
    float s[NR][4];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[nr][x] = 0.f;
    // S^T: lane (g8, t4) holds token rows g8 and g8 + 8, dims 64 cc + 16 t4 .. + 15
#pragma unroll
    for (int cc = 0; cc < KC; ++cc) {
      const uint4 a = lds16(kb + k_at<HD>(g8, cc * 4 + t4)), b = lds16(kb + k_at<HD>(g8 + 8, cc * 4 + t4));
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = to_h2(aw[i]), a2 = to_h2(aw[i] >> 16), a1 = to_h2(bw[i]), a3 = to_h2(bw[i] >> 16);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) mma(s[nr], a0, a1, a2, a3, qf[nr][cc * 4 + i][0], qf[nr][cc * 4 + i][1]);
      }
    }
    float ks, vs;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks), "=f"(vs) : "r"(kb + 32 * HD));
    bool grow = false, all = true;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) all = all && slot0 + 15 <= lim[nr][x] && slot0 > low[nr][x];
    all = __all_sync(0xffffffffu, all);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[nr][x] *= rs[nr][x & 1] * ks;
        if (!all) {
          const int slot = slot0 + g8 + (x >> 1) * 8;
          if (slot > lim[nr][x & 1] || slot <= low[nr][x & 1]) s[nr][x] = -INFINITY;
        }
        grow = grow || s[nr][x] > m[nr][x & 1] + LAZY;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float mx = fmaxf(s[nr][x], s[nr][x + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(mx, m[nr][x]);
          const float f = m[nr][x] == -INFINITY ? 0.f : ex2(m[nr][x] - mx);
          if (mx > m[nr][x]) {
            m[nr][x] = mx;
            l[nr][x] *= f;
#pragma unroll
            for (int j = 0; j < MT; ++j) { o[nr][j][x] *= f; o[nr][j][x + 2] *= f; }
          }
        }
    }
    // O is in units of vref; a block whose scale is within 2^6 of it goes in through P (at most 2^14)
    float ratio = 1.f;
    if (vs != vref) {
      if (vref == 0.f) vref = vs;
      else if (vs > vref * 64.f || (vs < vref * 0.015625f && vs > vref * 8.6736174e-19f)) {
        const float f = vref / vs;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[nr][j][x] *= f;
        vref = vs;
      } else ratio = vs / vref;
    }
    uint32_t pf[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float mm = m[nr][x & 1];
        e[x] = ex2(s[nr][x] - (mm == -INFINITY ? 0.f : mm));
        l[nr][x & 1] += e[x];
      }
      pf[nr][0] = transposed(pack_h2(e[0] * ratio, e[1] * ratio));
      pf[nr][1] = transposed(pack_h2(e[2] * ratio, e[3] * ratio));
    }
    // O^T: lane (g8, t4) holds tokens 2 t4, 2 t4 + 1 and the same + 8, dims HD / 8 * g8 ..
    uint32_t vw[4][HD / 32];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int r = 2 * t4 + (x & 1) + (x >> 1) * 8;
      if (HD == 128) {
        const uint4 v = lds16(vb + v_at<HD>(r, g8));
        vw[x][0] = v.x; vw[x][1] = v.y; vw[x][HD / 32 - 2] = v.z; vw[x][HD / 32 - 1] = v.w;
      } else {
        const uint2 v = lds8(vb + v_at<HD>(r, g8 >> 1) + (g8 & 1) * 8);
        vw[x][0] = v.x; vw[x][1] = v.y;
      }
      if (slot0 + 16 > it.hi) {                        // codes past the end may be anything, NaN included
        if (slot0 + r >= it.hi) {
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) vw[x][i] = 0;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const uint32_t x0 = __byte_perm(vw[0][i], vw[1][i], 0x5140), x1 = __byte_perm(vw[0][i], vw[1][i], 0x7362);
      const uint32_t y0 = __byte_perm(vw[2][i], vw[3][i], 0x5140), y1 = __byte_perm(vw[2][i], vw[3][i], 0x7362);
      const uint32_t a0 = to_h2(x0), a1 = to_h2(x0 >> 16), a2 = to_h2(y0), a3 = to_h2(y0 >> 16);
      const uint32_t b0 = to_h2(x1), b1 = to_h2(x1 >> 16), b2 = to_h2(y1), b3 = to_h2(y1 >> 16);
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        mma(o[nr][2 * i], a0, a1, a2, a3, pf[nr][0], pf[nr][1]);          // dims HD / 8 g8 + 4 i, + 1
        mma(o[nr][2 * i + 1], b0, b1, b2, b3, pf[nr][0], pf[nr][1]);      // + 2, + 3
      }
    }
  };

  float* mo = reinterpret_cast<float*>(smem + NW * STAGES * SB);        // [NW][ROWS][HD + 4]
  float* ml = mo + NW * ROWS * (HD + 4);                                 // [NW][ROWS][2]
  auto finish = [&](int64_t item_start, bool ends) {
    // sums over the lanes that share a row, then this warp's rows to shared memory
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v = l[nr][x];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        const int r = nr * 8 + 2 * t4 + x;
        if (g8 == 0) { ml[(w * ROWS + r) * 2] = m[nr][x]; ml[(w * ROWS + r) * 2 + 1] = v; }
        float* dst = mo + (w * ROWS + r) * (HD + 4) + g8 * (HD / 8);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          // tile j holds dims 2 j, 2 j + 1 of the lane's HD / 8
          *reinterpret_cast<float2*>(dst + 2 * j) = make_float2(o[nr][j][x] * vref, o[nr][j][x + 2] * vref);
        }
      }
    __syncthreads();
    const bool whole = ends && item_start >= first;
    float* part = p.part + ((int64_t)blockIdx.x * 2 + (item_start > first ? 1 : 0)) * ROWS * (HD + 2);
    const int per = p.rep * p.maps;
    for (int i = tid; i < ROWS / p.maps * (HD / 4); i += NT) {
      const int rr = i / (HD / 4) * p.maps, d = i % (HD / 4) * 4;      // first map's row
      if (it.rt * ROWS + rr >= it.rows) continue;
      float4 res = make_float4(0.f, 0.f, 0.f, 0.f);
      const int row = it.rt * ROWS + rr, tok = it.t0 + row / per, h = it.g * p.rep + row % per / p.maps;
      for (int map = 0; map < p.maps; ++map) {
        const int r = rr + map;
        float M = -INFINITY;
#pragma unroll
        for (int x = 0; x < NW; ++x) M = fmaxf(M, ml[(x * ROWS + r) * 2]);
        float L = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const float mm = ml[(x * ROWS + r) * 2];
          const float f = mm == -INFINITY ? 0.f : ex2(mm - M);
          const float4 v = *reinterpret_cast<const float4*>(mo + (x * ROWS + r) * (HD + 4) + d);
          L = fmaf(f, ml[(x * ROWS + r) * 2 + 1], L);
          a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
        }
        if (whole) {
          const float lam = p.maps == 2 ? p.lam[h] : 0.f;
          float f = L == 0.f ? 0.f : 1.f / L;
          if (p.maps == 2) f *= (map ? -lam : 1.f) / (1.f - lam + 1e-8f);
          res.x = fmaf(a.x, f, res.x); res.y = fmaf(a.y, f, res.y); res.z = fmaf(a.z, f, res.z); res.w = fmaf(a.w, f, res.w);
        } else {
          float2* dst = reinterpret_cast<float2*>(part + r * (HD + 2) + d);
          dst[0] = make_float2(a.x, a.y);
          dst[1] = make_float2(a.z, a.w);
          if (d == 0) *reinterpret_cast<float2*>(part + r * (HD + 2) + HD) = make_float2(M, L);
        }
      }
      if (whole) {
        T* out = (T*)p.out + ((int64_t)tok * p.H + h) * HD + d;
        union { T v[4]; uint2 raw; } u;
        u.v[0] = from_f<T>(res.x); u.v[1] = from_f<T>(res.y); u.v[2] = from_f<T>(res.z); u.v[3] = from_f<T>(res.w);
        *reinterpret_cast<uint2*>(out) = u.raw;
      }
    }
    if (ends && !whole && tid == 0)
      {
      const int64_t c0 = item_start / share;       // CTA and place of the item's first part
      p.joins[blockIdx.x] = make_int4(it.b, it.g, it.rt, (int)(2 * c0 + (item_start > c0 * share ? 1 : 0)));
    }
    __syncthreads();
  };

  load_rows();
  int tile = (int)(first - start);
  int stage = 0;
  for (int64_t pos = first; pos < last; ++pos) {
    issue((stage + STAGES - 1) % STAGES);
    cp_wait<STAGES - 1>();
    __syncwarp();
    if (live_bits >> stage & 1) compute(stage, (it.k0 + tile) * TILE + w * 16);
    __syncwarp();                                  // the slice is read before its slot is filled again
    stage = (stage + 1) % STAGES;
    if (++tile == it.nt || pos + 1 == last) {
      finish(start, tile == it.nt);
      if (pos + 1 < last) {
        start += it.nt;
        next_item<ROWS>(p, it);
        tile = 0;
        load_rows();
      }
    }
  }
  cp_wait<0>();
}

// Joins the parts of an item that ran over several CTAs: block = the CTA in which it ended.
template <typename T, int HD, int NR>
__global__ void __launch_bounds__(NT) join_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NR;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 j = p.joins[blockIdx.x];
  if (j.x < 0) return;
  Item it;
  set_sequence<ROWS>(p, it, j.x);
  it.g = j.y;
  it.rt = j.z;
  const int c0 = j.w >> 1, c1 = blockIdx.x, per = p.rep * p.maps;
  for (int i = threadIdx.x; i < ROWS / p.maps * (HD / 2); i += NT) {
    const int rr = i / (HD / 2) * p.maps, d = i % (HD / 2) * 2;
    const int row = it.rt * ROWS + rr;
    if (row >= it.rows) continue;
    float2 res = make_float2(0.f, 0.f);
    const int tok = it.t0 + row / per, h = it.g * p.rep + row % per / p.maps;
    for (int map = 0; map < p.maps; ++map) {
      float M = -INFINITY, L = 0.f;
      float2 a = make_float2(0.f, 0.f);
      for (int cta = c0; cta <= c1; ++cta) {
        const int slot = cta == c0 ? (j.w & 1) : 0;
        const float* part = p.part + (((int64_t)cta * 2 + slot) * ROWS + rr + map) * (HD + 2);
        const float2 v = *reinterpret_cast<const float2*>(part + d), s = *reinterpret_cast<const float2*>(part + HD);
        if (s.x == -INFINITY && s.y == 0.f) continue;
        const float mn = fmaxf(M, s.x), f = M == -INFINITY ? 0.f : ex2(M - mn), e = ex2(s.x - mn);
        a.x = a.x * f + v.x * e;
        a.y = a.y * f + v.y * e;
        L = L * f + s.y * e;
        M = mn;
      }
      const float lam = p.maps == 2 ? p.lam[h] : 0.f;
      float f = L == 0.f ? 0.f : 1.f / L;
      if (p.maps == 2) f *= (map ? -lam : 1.f) / (1.f - lam + 1e-8f);
      res.x = fmaf(a.x, f, res.x);
      res.y = fmaf(a.y, f, res.y);
    }
    T* out = (T*)p.out + ((int64_t)tok * p.H + h) * HD + d;
    out[0] = from_f<T>(res.x);
    out[1] = from_f<T>(res.y);
  }
}

template <typename T, int HD, int NR>
void launch_split(Params& p) {
  auto fn = split_kernel<T, HD, NR>;
  constexpr int SMEM = smem_bytes<HD, NR>();
  MAMF_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  fn<<<p.ctas, NT, SMEM, stream()>>>(p);
  MAMF_LAUNCH_CHECK();
  if (p.ctas == 1) return;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.ctas);
  cfg.blockDim = dim3(NT);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, HD, NR>, p));
}

}  // namespace pa

// q1, q2 (T, H, hd) bf16 or f16 packed queries -> (T, H, hd)
at::Tensor paged_attention(at::Tensor q1, c10::optional<at::Tensor> q2, c10::optional<at::Tensor> lam, at::Tensor ck,
                           at::Tensor cv, at::Tensor ks, at::Tensor vs, at::Tensor table, at::Tensor cu, at::Tensor lens,
                           int64_t max_new, int64_t window, double scale) {
  using namespace pa;
  TORCH_CHECK(q1.is_cuda() && q1.dim() == 3 && q1.device() == ck.device() && (q1.scalar_type() == at::kBFloat16 || q1.scalar_type() == at::kHalf),
              "paged_attention: bf16 or f16 queries (T, H, hd) on the cache's GPU");
  c10::cuda::CUDAGuard guard(q1.device());
  const int64_t T = q1.size(0), H = q1.size(1), hd = q1.size(2);
  Params p{};
  p.c = check_cache("paged_attention", Layer{ck, cv, ks, vs, table, cu, lens}, T, hd);
  TORCH_CHECK(H >= 1 && p.c.G >= 1 && H % p.c.G == 0, "paged_attention: ", H, " query heads over ", p.c.G, " KV heads");
  TORCH_CHECK(window >= 0 && max_new >= 0, "paged_attention: window and max_new must not be negative");
  q1 = rows16(q1);
  p.q1 = q1.data_ptr(); p.st1 = q1.stride(0); p.sh1 = q1.stride(1);
  if (q2.has_value()) {
    TORCH_CHECK(lam.has_value() && q2->is_cuda() && q2->device() == q1.device() && q2->sizes() == q1.sizes() && q2->scalar_type() == q1.scalar_type(),
                "paged_attention: q2 like q1, with lam");
    TORCH_CHECK(lam->is_cuda() && lam->device() == q1.device() && lam->scalar_type() == at::kFloat && lam->is_contiguous() && lam->numel() == H,
                "paged_attention: fp32 lam (H)");
    q2 = rows16(*q2);
    p.q2 = q2->data_ptr(); p.st2 = q2->stride(0); p.sh2 = q2->stride(1);
    p.lam = lam->data_ptr<float>();
  } else {
    TORCH_CHECK(!lam.has_value(), "paged_attention: lam without q2");
  }
  at::Tensor out = at::empty({T, H, hd}, q1.options());
  if (T == 0) return out;
  p.out = out.data_ptr();
  p.H = (int)H;
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.rep = (int)(H / p.c.G);
  p.maps = p.q2 ? 2 : 1;
  // one query row tile holds 8 rows, or 16 where some sequence can have more than 8
  const int nr = std::max<int64_t>(1, max_new) * p.rep * p.maps > 8 ? 2 : 1, rows = 8 * nr;
  const int64_t row_tiles = (std::max<int64_t>(1, std::min(max_new, T)) * p.rep * p.maps + rows - 1) / rows;
  const int64_t most = std::max<int64_t>(1, (int64_t)p.c.B * p.c.G * row_tiles * std::max<int64_t>(1, ((int64_t)p.c.W * p.c.page + TILE - 1) / TILE));
  p.ctas = (int)std::min<int64_t>(most, 3 * num_sms());
  const int64_t part = (int64_t)p.ctas * 2 * rows * (hd + 2);
  at::Tensor ws = at::empty({part + 4 * p.ctas}, q1.options().dtype(at::kFloat));
  p.joins = reinterpret_cast<int4*>(ws.data_ptr<float>());
  p.part = ws.data_ptr<float>() + 4 * p.ctas;
  auto go = [&](auto t) {
    using E = decltype(t);
    if (hd == 128) { if (nr == 1) launch_split<E, 128, 1>(p); else launch_split<E, 128, 2>(p); }
    else { if (nr == 1) launch_split<E, 64, 1>(p); else launch_split<E, 64, 2>(p); }
  };
  if (q1.scalar_type() == at::kBFloat16) go(__nv_bfloat16()); else go(__half());
  return out;
}

int64_t paged_attention_error() {
  int v = 0;
  MAMF_CUDA_CHECK(cudaMemcpyFromSymbol(&v, pa::g_err, sizeof(int)));
  if (v) {
    int z = 0;
    MAMF_CUDA_CHECK(cudaMemcpyToSymbol(pa::g_err, &z, sizeof(int)));
  }
  return v;
}

}  // namespace mamf
