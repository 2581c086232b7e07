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
// A CTA is 4 warps; warp w takes tokens 16 w .. 16 w + 15 of each tile through a ring of its own, filled by
// TMA (128-byte swizzle, one lane issues), and never waits for the other warps inside an item.  Its 16 tokens
// are the M rows of mma.m16n8k16 (f16 operands, fp32 sums): S^T = K Q^T and O^T = V^T P^T with up to 8 query
// rows as N, so 8 rows (4 heads of a group x 2 maps) fill the instruction; 16 rows take two.  e4m3 is exact
// in f16, and the rows of q are scaled by a power of two to [1, 2) first, which f16 holds exactly down to
// 2^-14 of a row's largest value.  P is rounded to f16 (11 bits; bf16 would keep 8).  The order of the head's
// dims in the products is free as long as both sides agree: a lane takes 16 adjacent bytes of K (and of V),
// so a fragment is one 16-byte read and no shuffles; so is the order of the 8 tokens of a fragment (`token`).
//
// 64 sequences of 300 to 8191 slots, 32 / 8 heads of 128, two maps (566 MB): 125 us, 4.5 TB/s, of which 8 us
// are the start and 6 the join.  One token on 131000 slots: 62.6 us.
#include "paged_split.cuh"

namespace mamf {
namespace pa {

using namespace split;

// Rows of a sequence and KV head above which the chunk kernel takes over.  This kernel and the chunk kernel, 16
// sequences of 2000-6000 slots, 32 / 8 heads, two maps: 24 rows 89 and 157 us, 32 rows 90 and 158, 64 rows 160 and
// 158; one map, 8 sequences of 8000, 16 / 4 heads: 32 rows 55 and 78, 64 rows 83 and 94 (of when the rule was set; since
// then 64 rows 84, and 80 rows 81 in the chunk kernel).
constexpr int FEW = 64;
constexpr int STEP = 16;                       // tokens of a warp per tile
constexpr int TILE = STEP * NW;                // tokens per tile
constexpr float LAZY = 8.f;                    // log2 by which a row may outgrow its reference maximum
constexpr float SLACK = 64.f;                  // value scales of up to this times O's unit are not looked at

struct Params : Attn {
  static constexpr bool SUMS = false;     // nobody asks for the rows' sums
  int ctas;
  float* part;        // [ctas][2][rows][HD + 2]: O (not divided), m, l
  int4* joins;        // [ctas]: {t0, rows, g | rt << 16, 2 c0 + place} of the item that ends in this CTA after it
                      // began in CTA c0 (its part there is in `place`), or {-1, ..}
};

// four e4m3 codes -> the first two and the last two as f16 (exact)
__device__ __forceinline__ void to_h4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void tma_lines(uint32_t dst, const CUtensorMap* map, uint32_t bar, int line) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(line) : "memory");
}
template <int HD> constexpr int stage_bytes() { return 2 * STEP * HD; }
constexpr int ST = 3;                          // tiles of a warp's ring
// resident CTAs per SM: the latency of a warp's chain (products, exponentials, products) is hidden by other
// warps, so there are as many as the registers of a row tile allow without spills (128, 168 or 255)
template <int HD, int NR> constexpr int residents() { return NR == 1 ? 4 : HD == 64 ? 3 : 2; }
template <int HD, int NR> constexpr int merge_words() { return NR * (HD / 4 + 4); }      // of a lane
template <int HD, int NR> constexpr int smem_bytes() {
  return 1024 + NW * ST * stage_bytes<HD>() + 32 * 4 * merge_words<HD, NR>();
}

// The token of row r (0..7) of a fragment, and where TMA's 128-byte swizzle puts 16-byte chunk c of token n
// (0..15) of a slice: chunk index xor line & 7, a line being one token of 128 dims or two of 64.  The orders
// make the lanes of each phase of a shared-memory read hit every bank once: for K two rows r = 2 i, 2 i + 1 at
// four chunks, for V the rows 2 i (then 2 i + 1) of four i at two chunks.
template <int HD> __device__ __forceinline__ int token(int r) {
  return HD == 128 ? (int)(0x36147250u >> (4 * r) & 7) : (int)(0x65742130u >> (4 * r) & 7);
}
template <int HD> __device__ __forceinline__ int chunk_at(int n, int c) {
  if (HD == 128) return n * 128 + ((c ^ (n & 7)) << 4);
  return (n >> 1) * 128 + ((((n & 1) * 4 + c) ^ (n >> 1 & 7)) << 4);
}

template <typename T, int HD, int NR>
__global__ void __launch_bounds__(NT, residents<HD, NR>()) split_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap map_k,
                                                      const __grid_constant__ CUtensorMap map_v) {
  constexpr int ROWS = 8 * NR;
  constexpr int KC = HD / 64;                    // 16-byte reads of a K row per lane
  constexpr int MT = HD / 16;                    // 16-dim tiles of O^T
  constexpr int SB = stage_bytes<HD>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[NW][ST];
  __shared__ int64_t s_pre[NT / 32];
  __shared__ int64_t s_begin;
  __shared__ int s_b, s_cut;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  const Cache& c = p.c;
  asm volatile("griddepcontrol.launch_dependents;");      // the join kernel waits for this grid's end by itself

  // ---- this CTA's share [first, last) of the list of tiles ----
  const int chunk = (c.B + NT - 1) / NT;
  int64_t mine = 0;
  bool broken = false;                              // offsets out of order: nothing is done here
  for (int i = 0; i < chunk; ++i) {
    const int b = tid * chunk + i;
    if (b < c.B) {
      mine += tiles_of<ROWS, TILE>(p, b);
      broken = broken || !in_order(c, b);
    }
  }
  broken = __any_sync(0xffffffffu, broken);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_pre[w] = broken ? 1LL << 60 : incl;
  if (tid == 0) { s_b = -1; s_cut = 0; }
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
      const int64_t n = tiles_of<ROWS, TILE>(p, b);
      if (first < at + n) break;
      at += n;
    }
    s_b = b;
    s_begin = at;
  }
  __syncthreads();
  if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
  // rows before the first and past the last sequence
  {
    const int64_t row = (int64_t)p.H * HD;
    const int64_t front = c.B > 0 ? min(max(0, c.cu[0]), c.T) * row : 0, end = c.B > 0 ? max(0, c.cu[c.B]) * row : 0;
    for (int64_t i = (int64_t)blockIdx.x * NT + tid; i < front; i += (int64_t)gridDim.x * NT) ((T*)p.out)[i] = from_f<T>(0.f);
    for (int64_t i = end + (int64_t)blockIdx.x * NT + tid; i < c.T * row; i += (int64_t)gridDim.x * NT)
      ((T*)p.out)[i] = from_f<T>(0.f);
  }
  if (first >= last || total >> 60) return;

  Item it;                                          // of the tile being computed
  set_sequence<ROWS, TILE>(p, it, s_b);
  int64_t start = s_begin;                          // list position of the item's first tile
  while (first >= start + it.nt) { start += it.nt; next_item<ROWS, TILE>(p, it); }

  // ---- ring: the issue side runs ST - 1 tiles ahead ----
  const uint32_t ring = su32(smem) + w * ST * SB, bar = su32(bars[w]);
  if (lane < ST) tc5::bar_init(&bars[w][lane], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  Item is = it;
  int to_issue = (int)(last - first), issued = 0, waited = 0;
  int is_left = it.nt - (int)(first - start);                        // tiles of the item still to be looked up
  int is_slot = (it.k0 + (int)(first - start)) * TILE + w * STEP;     // the warp's first token of the tile
  const int* is_table = c.table + (int64_t)is.b * c.W;
  // the page of the warp's 16 tokens of a tile: -2 nothing to see there, -1 not a page of the pool
  int pg;
  auto look_up = [&]() {
    pg = -2;
    if (is_slot < is.hi && is_slot + STEP > is.lo) {
      const int j = is_slot >> c.shift;
      pg = j < c.W ? is_table[j] : -1;
    }
  };
  look_up();
  // scales of the tiles in flight, newest last; a K scale of 0 marks tokens that are not there
  float ksr[ST], vsr[ST];
  bool ok = true;
  auto issue = [&](uint32_t stage_at, uint32_t bar_at) {
#pragma unroll
    for (int i = 0; i + 1 < ST; ++i) { ksr[i] = ksr[i + 1]; vsr[i] = vsr[i + 1]; }
    ksr[ST - 1] = vsr[ST - 1] = 0.f;
    if (to_issue <= 0) return;
    ++issued;
    const bool there = (unsigned)pg < (unsigned)c.P;
    const int blk = pg * c.G + is.g;
    if (there) {
      ksr[ST - 1] = c.ks[blk];
      vsr[ST - 1] = c.vs[blk];
    }
    if (lane == 0) {
      if (there) {
        const int token = (blk << c.shift) + (is_slot & (c.page - 1)), line = HD == 128 ? token : token >> 1;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar_at), "r"(SB) : "memory");
        tma_lines(stage_at, &map_k, bar_at, line);
        tma_lines(stage_at + STEP * HD, &map_v, bar_at, line);
      } else {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_at) : "memory");
        if (pg != -2) record(ERR_PAGE);
      }
    }
    if (--to_issue > 0) {
      is_slot += TILE;
      if (--is_left == 0) {
        next_item<ROWS, TILE>(p, is);
        is_left = is.nt;
        is_slot = is.k0 * TILE + w * STEP;
        is_table = c.table + (int64_t)is.b * c.W;
      }
      look_up();
    }
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(ring + s * SB, bar + s * 8);

  // ---- state of the current item ----
  uint32_t qf[NR][KC * 4][2];
  float rs[NR][2];                        // score factor of rows 2 t4, 2 t4 + 1
  int lim[NR][2], low[NR][2];             // slots (low, lim] that the row sees
  int all_lo = 0, all_hi = 0;             // slots [all_lo, all_hi] that every row sees
  // m: a row's running maximum of the scores, which l is kept in.  O is kept in units of 2^(m + off), off a whole number
  // that brings m + off to the row's running maximum of score + log2 of the value scale: what a page of other values
  // holds takes no bits from a row that gives it no weight.
  float m[NR][2], l[NR][2], o[NR][MT][4];
  int noff[NR][2];                        // -off, as what it adds to the exponent bits of a scale
  // 2^-off times a scale, between 0 and 2^126: keys of no weight may have any scale
  auto ratio_of = [&](float vs, int nr, int x) {
    return __int_as_float(__viaddmin_s32_relu((int)__float_as_uint(vs), noff[nr][x], 253 << 23));
  };
  auto load_rows = [&]() {
    const int per = p.rep * p.maps, at0 = it.len - it.n;
    all_hi = min(it.len - 1, at0 + it.rt * ROWS / per);
    all_lo = p.window > 0 ? at0 + min(it.n - 1, (it.rt * ROWS + ROWS - 1) / per) - p.window + 1 : 0;
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
        m[nr][x] = NONE;
        l[nr][x] = 0.f;
        noff[nr][x] = 0;
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[nr][j][x] = 0.f;
    }
  };

  // rows of this lane in the fragments: token tk (K) and tv[0], tv[1] (V), and the same + 8, which is
  // 8 lines (or 4, with bit 2 of the chunk flipped) further on; 64 dims on is bit 2 of the chunk
  const int tk = token<HD>(g8), tv[2] = {token<HD>(2 * t4), token<HD>(2 * t4 + 1)};
  const uint32_t k_off = chunk_at<HD>(tk, t4);
  const uint32_t v_off[2] = {(uint32_t)chunk_at<HD>(tv[0], HD == 128 ? g8 : g8 >> 1) + (HD == 128 ? 0 : (g8 & 1) * 8),
                             (uint32_t)chunk_at<HD>(tv[1], HD == 128 ? g8 : g8 >> 1) + (HD == 128 ? 0 : (g8 & 1) * 8)};
  auto plus8 = [](uint32_t a) { return HD == 128 ? a + 1024 : (a + 512) ^ 64; };
  auto scores = [&](uint32_t kb, float ks, int slot0, float (&s)[NR][4]) {
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[nr][x] = 0.f;
    // S^T: tokens tk and tk + 8, dims 64 cc + 16 t4 .. + 15
#pragma unroll
    for (int cc = 0; cc < KC; ++cc) {
      const uint32_t at = (kb + k_off) ^ (cc * 64);
      const uint4 a = lds16(at), b = lds16(plus8(at));
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0, a1, a2, a3;
        to_h4(aw[i], a0, a2);
        to_h4(bw[i], a1, a3);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) mma(s[nr], a0, a1, a2, a3, qf[nr][cc * 4 + i][0], qf[nr][cc * 4 + i][1]);
      }
    }
    const bool all = slot0 + STEP - 1 <= all_hi && slot0 >= all_lo;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[nr][x] *= rs[nr][x & 1] * ks;
        if (!all) {
          const int slot = slot0 + tk + (x >> 1) * 8;
          if (slot > lim[nr][x & 1] || slot <= low[nr][x & 1]) s[nr][x] = -INFINITY;
        }
      }
  };
  auto raise = [&](float (&s)[NR][4], float vs) {
    bool grow = false;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        grow = grow || fmaxf(s[nr][x], s[nr][x + 2]) > m[nr][x] + LAZY || ratio_of(vs, nr, x) > SLACK;
    if (!__any_sync(0xffffffffu, grow)) return;
    const float lv = (float)((int)(__float_as_uint(vs) >> 23) - 127);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float mx = fmaxf(s[nr][x], s[nr][x + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m0 = m[nr][x], off = (float)(-(noff[nr][x] >> 23)), m1 = fmaxf(m0, mx);
        const float to = mx + lv > m0 + off ? mx + lv : m0 + off;
        const float u1 = fminf(fmaxf(rintf(to - m1), -126.f), 126.f);
        const float f = ex2((m0 - m1) + (off - u1));
        l[nr][x] *= ex2(m0 - m1);
        m[nr][x] = m1;
        noff[nr][x] = -((int)u1 << 23);
#pragma unroll
        for (int j = 0; j < MT; ++j) { o[nr][j][x] *= f; o[nr][j][x + 2] *= f; }
      }
  };
  // P V of one tile.  The weights that enter it are at most 2^LAZY * SLACK.
  auto values = [&](uint32_t vb, float vs, int slot0, float (&s)[NR][4]) {
    uint32_t pf[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        e[x] = ex2(s[nr][x] - m[nr][x & 1]);
        l[nr][x & 1] += e[x];
        e[x] *= ratio_of(vs, nr, x & 1);
      }
      pf[nr][0] = transposed(pack_h2(e[0], e[1]));
      pf[nr][1] = transposed(pack_h2(e[2], e[3]));
    }
    // O^T: tokens tv[0], tv[1] and the same + 8, dims HD / 8 * g8 ..
    uint32_t vw[4][HD / 32];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t at = x < 2 ? vb + v_off[x] : plus8(vb + v_off[x - 2]);
      if (HD == 128) {
        const uint4 v = lds16(at);
        vw[x][0] = v.x; vw[x][1] = v.y; vw[x][HD / 32 - 2] = v.z; vw[x][HD / 32 - 1] = v.w;
      } else {
        const uint2 v = lds8(at);
        vw[x][0] = v.x; vw[x][1] = v.y;
      }
    }
    if (slot0 + 16 > it.hi) {                          // codes past the end may be anything, NaN included
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (slot0 + tv[x & 1] + (x >> 1) * 8 >= it.hi) {
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) vw[x][i] = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
      to_h4(__byte_perm(vw[0][i], vw[1][i], 0x5140), a0, a1);
      to_h4(__byte_perm(vw[2][i], vw[3][i], 0x5140), a2, a3);
      to_h4(__byte_perm(vw[0][i], vw[1][i], 0x7362), b0, b1);
      to_h4(__byte_perm(vw[2][i], vw[3][i], 0x7362), b2, b3);
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        mma(o[nr][2 * i], a0, a1, a2, a3, pf[nr][0], pf[nr][1]);          // dims HD / 8 g8 + 4 i, + 1
        mma(o[nr][2 * i + 1], b0, b1, b2, b3, pf[nr][0], pf[nr][1]);      // + 2, + 3
      }
    }
  };

  // Warps 3, 2, 1 pass their joined state on through shared memory, lane by lane; warp 0 writes the result.
  float* merge = reinterpret_cast<float*>(smem + NW * ST * SB) + lane;
  auto finish = [&](int64_t item_start, bool ends) {
    float unit[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) unit[nr][x] = __int_as_float((127 << 23) - noff[nr][x]);
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[nr][j][x] *= unit[nr][x & 1];
#pragma unroll 1
    for (int turn = NW - 1; turn >= 0; --turn) {
      if (w == turn && turn < NW - 1) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float mm = merge[(nr * 4 + x) * 32], M = fmaxf(m[nr][x], mm);
            const float a = ex2(m[nr][x] - M), b = ex2(mm - M);
            m[nr][x] = M;
            l[nr][x] = fmaf(l[nr][x], a, merge[(nr * 4 + 2 + x) * 32] * b);
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
              for (int z = x; z < 4; z += 2) o[nr][j][z] = fmaf(o[nr][j][z], a, merge[(NR * 4 + (nr * MT + j) * 4 + z) * 32] * b);
          }
      }
      if (w == turn && turn > 0) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
          for (int x = 0; x < 2; ++x) { merge[(nr * 4 + x) * 32] = m[nr][x]; merge[(nr * 4 + 2 + x) * 32] = l[nr][x]; }
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) merge[(NR * 4 + (nr * MT + j) * 4 + x) * 32] = o[nr][j][x];
        }
      }
      if (turn > 0) __syncthreads();
    }
    if (w == 0) {
      const bool whole = ends && item_start >= first, cut = *(volatile int*)&s_cut != 0;
      float* part = p.part + ((int64_t)blockIdx.x * 2 + (item_start > first ? 1 : 0)) * ROWS * (HD + 2);
      const int per = p.rep * p.maps;
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        float f0[2];                                     // 1 / sum over the row's lanes
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float M = m[nr][x];
          float L = l[nr][x];
          L += __shfl_xor_sync(0xffffffffu, L, 4);
          L += __shfl_xor_sync(0xffffffffu, L, 8);
          L += __shfl_xor_sync(0xffffffffu, L, 16);
          if (cut) L = -1.f;                             // in a part: the join writes zeros
          f0[x] = cut || L == 0.f ? 0.f : 1.f / L;
          const int r = nr * 8 + 2 * t4 + x;
          if (!whole) {
            float* dst = part + r * (HD + 2);
#pragma unroll
            for (int j = 0; j < MT; ++j)
              *reinterpret_cast<float2*>(dst + g8 * (HD / 8) + 2 * j) = make_float2(o[nr][j][x], o[nr][j][x + 2]);
            if (g8 == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(M, L);
          }
        }
        if (!whole) continue;
        // rows 2 t4 and 2 t4 + 1 are two heads, or the two maps of one
        const int row = it.rt * ROWS + nr * 8 + 2 * t4;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (row + x >= it.rows || (x == 1 && p.maps == 2)) continue;
          const int tok = it.t0 + (row + x) / per, h = it.g * p.rep + (row + x) % per / p.maps;
          float wa = f0[x], wb = 0.f;
          if (p.maps == 2) {
            const float lam = p.lam[h], den = 1.f / (1.f - lam + 1e-8f);
            wa *= den;
            wb = -lam * den * f0[1];
          }
          T* out = (T*)p.out + ((int64_t)tok * p.H + h) * HD + g8 * (HD / 8);
#pragma unroll
          for (int j = 0; j < MT; j += 4) {
            Vec16<T> v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float a0 = o[nr][j + k][x] * wa, a1 = o[nr][j + k][x + 2] * wa;
              v.v[2 * k] = from_f<T>(p.maps == 2 ? fmaf(o[nr][j + k][1], wb, a0) : a0);
              v.v[2 * k + 1] = from_f<T>(p.maps == 2 ? fmaf(o[nr][j + k][3], wb, a1) : a1);
            }
            st16(out + 2 * j, v);
          }
        }
      }
      if (ends && !whole && lane == 0) {
        const int64_t c0 = item_start / share;       // CTA and place of the item's first part
        p.joins[blockIdx.x] = make_int4(it.t0, it.rows, it.g | it.rt << 16, (int)(2 * c0 + (item_start > c0 * share ? 1 : 0)));
      }
    }
    __syncthreads();
  };

  load_rows();
  int tiles = it.nt - (int)(first - start);                           // of the item, still to be done
  int slot0 = (it.k0 + (int)(first - start)) * TILE + w * STEP;
  uint32_t here = ring, bar_here = bar, phase = 0, there = ring + (ST - 1) * SB, bar_there = bar + (ST - 1) * 8;
  for (int left = (int)(last - first); left > 0; --left) {
    if (ok) {
      issue(there, bar_there);
      ok = wait_tile(bar_here, phase, p.wait);
      waited += ok;
      if (!ok) s_cut = 1;                          // this item's rows and the next ones' are zeros
    }
    if (ok && ksr[0] != 0.f) {
      float s[NR][4];
      scores(here, ksr[0], slot0, s);
      raise(s, vsr[0]);
      values(here + STEP * HD, vsr[0], slot0, s);
    }
    __syncwarp();                                  // the tile is read before its place is filled again
    there = here;
    bar_there = bar_here;
    here += SB;
    bar_here += 8;
    if (here == ring + ST * SB) { here = ring; bar_here = bar; phase ^= 1; }
    slot0 += TILE;
    if (--tiles == 0 || left == 1) {
      finish(start, tiles == 0);
      if (left > 1) {
        start += it.nt;
        next_item<ROWS, TILE>(p, it);
        tiles = it.nt;
        slot0 = it.k0 * TILE + w * STEP;
        load_rows();
      }
    }
  }
  // after a wait that ran out: the copies that are still under way into this CTA's memory
  for (; waited < issued; ++waited) drain_tile(bar + waited % ST * 8, (uint32_t)(waited / ST & 1));
}

// All tokens of a cache tensor as lines of 128 bytes, a box of 16 tokens (they are adjacent in their page).
static CUtensorMap lines_map(const uint8_t* base, int64_t tokens, int hd) {
  CUtensorMap m;
  cuuint64_t gd[2] = {128, (cuuint64_t)(tokens * hd / 128)};
  cuuint64_t gs[1] = {128};
  cuuint32_t bx[2] = {128u, (cuuint32_t)(16 * hd / 128)}, es[2] = {1, 1};
  const CUresult r = tc5_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), gd, gs, bx, es,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "paged_attention: cuTensorMapEncodeTiled failed: ", (int)r);
  return m;
}

template <typename T, int HD, int NR>
void launch_split(const Params& p, const CUtensorMap& mk, const CUtensorMap& mv) {
  auto fn = split_kernel<T, HD, NR>;
  constexpr int SMEM = smem_bytes<HD, NR>();
  static bool set[64] = {};                              // by device; the attribute stays
  int dev = 0;
  MAMF_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    MAMF_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) set[dev] = true;
  }
  fn<<<p.ctas, NT, SMEM, stream()>>>(p, mk, mv);
  MAMF_LAUNCH_CHECK();
  launch_join<T, HD, NR>(p);
}

}  // namespace pa

static long long g_wait_limit = paged::WAIT_CYCLES;
long long paged::attention_wait_limit() { return g_wait_limit; }

// Sets the cycles after which the waits of later calls give up (negative: at once), for tests of what follows;
// returns the number before.
int64_t paged_attention_wait_limit(int64_t cycles) {
  const int64_t had = g_wait_limit;
  g_wait_limit = cycles;
  return had;
}

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
  TORCH_CHECK(std::isfinite((float)(scale * 1.4426950408889634)), "paged_attention: a finite scale, got ", scale);
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
  TORCH_CHECK(p.c.P >= 1, "paged_attention: a pool without pages");
  p.out = out.data_ptr();
  p.H = (int)H;
  p.window = (int)std::min<int64_t>(window, 1LL << 30);
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.wait = g_wait_limit;
  p.rep = (int)(H / p.c.G);
  p.maps = p.q2 ? 2 : 1;
  TORCH_CHECK(T * H < (1LL << 31), "paged_attention: sizes");
  // Sequences of up to FEW rows go to the split kernel, longer runs of tokens to the chunk kernel; where all
  // have the same number of tokens one of them does everything.
  const int64_t most_rows = std::max<int64_t>(1, std::min(max_new, T)) * p.rep * p.maps;
  p.chunked = most_rows > FEW && p.c.B > 0;
  const bool alone = p.chunked && T == p.c.B * max_new;
  p.few = alone ? 0 : (int)std::min<int64_t>(most_rows, FEW);
  if (p.chunked) paged_chunk_attention(p, (int)hd, q1.scalar_type() == at::kBFloat16);
  if (alone) return out;
  // one query row tile holds 8 rows, or 16 where a sequence can have more than 8
  const int nr = p.few > 8 ? 2 : 1, rows = 8 * nr;
  const int64_t row_tiles = (p.few + rows - 1) / rows;
  const int64_t most = std::max<int64_t>(1, (int64_t)p.c.B * p.c.G * row_tiles * std::max<int64_t>(1, ((int64_t)p.c.W * p.c.page + TILE - 1) / TILE));
  p.ctas = (int)std::min<int64_t>(most, (nr == 1 ? residents<128, 1>() : hd == 64 ? residents<64, 2>() : residents<128, 2>()) * num_sms());
  const int64_t part = (int64_t)p.ctas * 2 * rows * (hd + 2);
  at::Tensor ws = at::empty({part + 4 * p.ctas}, q1.options().dtype(at::kFloat));
  p.joins = reinterpret_cast<int4*>(ws.data_ptr<float>());
  p.part = ws.data_ptr<float>() + 4 * p.ctas;
  TORCH_CHECK((int64_t)p.c.P * p.c.G * p.c.page < (1LL << 31), "paged_attention: a pool of 2^31 tokens and heads or more");
  const int64_t tokens = (int64_t)p.c.P * p.c.G * p.c.page;
  const CUtensorMap mk = lines_map(p.c.k, tokens, (int)hd), mv = lines_map(p.c.v, tokens, (int)hd);
  auto go = [&](auto t) {
    using E = decltype(t);
    if (hd == 128) { if (nr == 1) launch_split<E, 128, 1>(p, mk, mv); else launch_split<E, 128, 2>(p, mk, mv); }
    else { if (nr == 1) launch_split<E, 64, 1>(p, mk, mv); else launch_split<E, 64, 2>(p, mk, mv); }
  };
  if (q1.scalar_type() == at::kBFloat16) go(__nv_bfloat16()); else go(__half());
  return out;
}

int64_t paged_attention_error(bool clear) {
  return paged::take_code(split::g_err, clear) | paged::take_code(split::g_wait_err, clear) | paged::paged_chunk_error(clear);
}

}  // namespace mamf
