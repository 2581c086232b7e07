// Attention over the paged 4-bit cache (layout in paged4.cuh), for few query rows per KV head: single tokens and short
// runs of tokens; with the weights that each slot receives, where they are asked for.
//
//   S = scale q . k,  P = 2^(S log2 e - r),  O = sum P v / sum P,   causal, optional window;
//   differential: (O1 - lam O2) / (1 - lam + 1e-8);   mass[slot] += sum over rows and maps of P / sum P
//
// The work is the list of (sequence, KV head, row tile) items, each a run of 128-token tiles; the grid's CTAs take equal
// contiguous shares of that list, so one long sequence fills the GPU as well as many short ones.  An item that ends in
// another CTA than it began in leaves partial (r, l, O) in a workspace and a second small kernel joins them in order
// (results do not depend on timing).
//
// A CTA is 4 warps; warp w takes tokens 32 w .. 32 w + 31 of each tile, which are two blocks of the cache, through a ring
// of its own: one bulk copy for both, or one a block where a page is one block, issued by one lane.  It never waits for the
// other warps inside an item.  A block's 16 tokens are the M rows of mma.m16n8k16 (f16 operands, fp32 sums): S^T = K Q^T and O^T = V^T P^T with up to 8 query rows
// as N; 16 rows take two.  A code becomes its f16 value in three instructions for two dims, exactly, so the products are
// those of the stored values; the rows of q are scaled by a power of two to [1, 2) first, which f16 holds exactly down to
// 2^-14 of a row's largest value.  P is rounded to f16 (11 bits; bf16 would keep 8) at up to 2^15, so that weights down to
// 2^-21 of a row's largest keep all of their bits, whatever values they are given to; f16 results of short runs are 2.7e-4 from
// 64 bits, 2.1e-4 with fp32 weights, and in bf16 the result's own rounding hides it.  The order of the head's dims in the
// products is free as long as both sides agree: a lane takes 16 adjacent bytes of a key's codes and 8 of a value's.
//
// Received weights: the scores of up to 16 rows are left in a workspace, 4 bytes a row and slot, for at most twice
// the slots of the pool (a slot of the cache has 76 or 148 bytes), and a last kernel turns them into weights with each row's
// joined sum; longer runs of tokens have them computed from the keys once more (paged4_attn_tc.cu).
//
// What bounds it: instructions.  64 sequences of 4096 slots, 32 / 8 heads of 128, two maps (302 MB): 97 us, where reading
// takes 46; 65% of the issue slots, half of the ALU's (decoding), DRAM 39%, tensor 17%, 14 warps an SM on average.
#include "paged4.cuh"
#include "paged_split.cuh"

#include <cooperative_groups.h>

namespace mamf {
namespace pa4 {

namespace cg = cooperative_groups;

using namespace split;
using namespace paged4;

// Rows of a sequence and KV head above which the chunk kernel takes over.  us on this kernel and on that one, 8 sequences of
// 8000 slots: one map of 16 / 4 heads, 48 rows 58 and 72, 64 rows 77 and 87, 80 rows 125 and 87; two maps of 32 / 8, 64 rows
// 128 and 194, 96 rows 185 and 195, 128 rows 239 and 196.
constexpr int FEW = 64;
constexpr int NB = 2, STEP = 16 * NB;          // blocks and tokens of a warp per tile
constexpr int TILE = STEP * NW;                // tokens per tile
constexpr float LIFT = 7.f, LAZY = 8.f;        // a row's largest weight is 2^LIFT when its reference is set, and may outgrow it
constexpr int MOST = 8;                        // CTAs of a cluster
// Each item gets a cluster of its own where all of these fit on the GPU at once and a CTA has at most SHORT tiles, of the
// longest sequence that the table has room for (the host does not know the lengths): no list to be shared, no second
// kernel.  Clusters and list, one map of 16 / 4 heads, us a call: 1 sequence of 700 slots 10.7 and 12.8, of 4000 14.7 and
// 14.8, of 8000 20.9 and 16.8; 16 of 700 13.8 and 16.5, of 4000 22.3 and 25.1, of 8000 33.3 and 35.0; 64 of 700 20.6 and
// 22.9, of 8000 103 and 99.  At 8000 slots it takes the list, which is right for few sequences and for very many.
constexpr int SHORT = 4;
// Rows whose scores are left for the received weights, at most: 4 rows 36 us and, computed from the keys once more, 88, 16 rows
// 45 and 131 (8 sequences of 8000 slots); 16 rows, two maps, 64 of 4000, 190 and 957.  More would take more than the cache.
constexpr int KEEP = 16;

// A sequence's scores: [G][n][stride] from slot `lo` on, behind those of `start` slots; start < 0: not kept.
struct Place { int64_t start; int lo, n; };

struct Params : Attn4 {
  static constexpr bool SUMS = true;      // the rows' sums may be asked for
  int ctas;
  float* part;        // [ctas][2][rows][HD + 2]: O (not divided), r, l
  int4* joins;        // [ctas]: {t0, rows, g | rt << 16, 2 c0 + place} of the item that ends in this CTA after it
                      // began in CTA c0 (its part there is in `place`), or {-1, ..}
  float* scores;      // scores (log2) of up to `stride` rows of a slot, where weights are asked for
  const Place* places;                     // [B] where a sequence's scores are; null: at b cap, of all slots
  int64_t cap;        // slots that a sequence can have
  int stride;
};

// Slots in front of slot 0's scores of a sequence and KV head (less than 0 where slots in front of `lo` are left out), or NOT_KEPT.
constexpr int64_t NOT_KEPT = -(1LL << 62);
__device__ __forceinline__ int64_t scores_of(const Params& p, int b, int g) {
  if (!p.places) return ((int64_t)b * p.c.G + g) * p.cap;
  const Place at = p.places[b];
  return at.start < 0 ? NOT_KEPT : at.start * p.c.G + (int64_t)g * at.n - at.lo;
}

__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

// mma() onto zeros
__device__ __forceinline__ void mma_new(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

constexpr int ST = 2;                          // tiles of a warp's ring
// resident CTAs per SM: the latency of a warp's chain (products, exponentials, products) is hidden by other
// warps, so there are as many as the registers of a row tile allow without spills (128, 168 or 255)
template <int HD, int NR> constexpr int residents() { return NR == 1 ? 4 : HD == 64 ? 3 : 2; }
template <int HD, int NR> constexpr int merge_words() { return NR * (HD / 4 + 4); }      // of a lane
template <int HD, int NR, bool ALONE> constexpr int smem_bytes() {
  return 1024 + NW * ST * NB * BLOCK<HD> + 32 * 4 * merge_words<HD, NR>() + (ALONE ? 8 * NR * (HD + 2) * 4 : 0);
}

// ALONE: a cluster of CTAs for each item shares its tiles and joins its parts through distributed shared memory.  Else
// contiguous shares of all items' tiles, and the join kernel.
template <typename T, int HD, int NR, bool ALONE>
__global__ void __launch_bounds__(NT, residents<HD, NR>()) split_kernel(const __grid_constant__ Params p) {
  constexpr int ROWS = 8 * NR;
  constexpr int KW = HD / 32;                    // words of a K row per lane, and of the parameters of a row's two halves
  constexpr int VW = HD / 64;                    // words of a V row per lane
  constexpr int MT = HD / 16;                    // 16-dim tiles of O^T
  constexpr int SB = NB * BLOCK<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[NW][ST];
  __shared__ int64_t s_pre[NT / 32];
  __shared__ int64_t s_begin;
  __shared__ int s_b, s_cut;
  // What the warps need at an item's ends only, and so keep out of registers: its description for the tiles being computed
  // and for those being fetched, and the slots (x, y] that each of its rows sees.
  __shared__ Item s_item[NW][2];
  __shared__ int2 s_sees[NW][8 * NR];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
  const Cache4& c = p.c;
  asm volatile("griddepcontrol.launch_dependents;");      // the join kernel waits for this grid's end by itself

  const int rank = ALONE ? (int)cg::this_cluster().block_rank() : 0;
  int64_t first, last, share = 1;                   // this CTA's tiles, of the item or of the list
  bool nothing;
  if constexpr (ALONE) {
    const int b = blockIdx.z, g = blockIdx.y % c.G;
    bool broken = false;
    for (int i = tid; i < c.B; i += NT) broken = broken || !in_order(c, i);
    if (tid == 0) s_cut = 0;
    broken = __syncthreads_or(broken);
    Item x;
    const bool mine = !broken && set_sequence<ROWS, TILE>(p, x, b);
    first = last = 0;
    nothing = !mine;
    if (mine) {
      x.g = g;
      x.rt = blockIdx.y / c.G;
      nothing = x.rt * ROWS >= x.rows;
      if (!nothing) {
        set_range<ROWS, TILE>(p, x);
        const int C = gridDim.x, per = (x.nt + C - 1) / C;
        first = min(x.nt, rank * per);
        last = min(x.nt, rank * per + per);
        s_item[w][0] = x;
      }
      if (tid == 0 && rank == 0 && cached_length(c, c.lens[b]) != c.lens[b]) record(ERR_LENGTH);
    } else if (broken || c.cu[b + 1] > c.cu[b]) {   // offsets out of order anywhere: zeros everywhere; more rows than were said: its rows
      const int64_t row = (int64_t)p.H * HD, C = gridDim.x;
      const int64_t from = broken ? 0 : c.cu[b], to = broken ? c.T : c.cu[b + 1];
      const int64_t step = C * NT * gridDim.y * (broken ? c.B : 1);
      for (int64_t i = from * row + ((int64_t)((broken ? b : 0) * gridDim.y + blockIdx.y) * C + rank) * NT + tid; i < to * row; i += step) ((T*)p.out)[i] = from_f<T>(0.f);
      if (p.lse)
        for (int64_t i = from * p.H * p.maps + tid; i < to * p.H * p.maps; i += NT) p.lse[i] = INFINITY;
      if (tid == 0) record(ERR_LENGTH);
    }
    if (broken) return;
  } else {
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
  share = (total + p.ctas - 1) / p.ctas;
  first = blockIdx.x * share;
  last = min(total, first + share);
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
  nothing = first >= last || total >> 60;
  }
  // rows before the first and past the last sequence
  {
    const int64_t row = (int64_t)p.H * HD;
    const int64_t front = c.B > 0 ? min(max(0, c.cu[0]), c.T) * row : 0, end = c.B > 0 ? max(0, c.cu[c.B]) * row : 0;
    const int64_t at = (((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * NT + tid, step = (int64_t)gridDim.x * gridDim.y * gridDim.z * NT;
    for (int64_t i = at; i < front; i += step) ((T*)p.out)[i] = from_f<T>(0.f);
    for (int64_t i = end + at; i < c.T * row; i += step) ((T*)p.out)[i] = from_f<T>(0.f);
  }

  if (nothing) return;                              // the CTAs of a cluster agree on this

  Item& it = s_item[w][0];                          // of the tile being computed
  Item& is = s_item[w][1];                          // of the next tile to be fetched
  int done = 0;                                     // tiles of the first item that are other CTAs'
  int64_t start = 0;                                // list position of the item's first tile
  if constexpr (ALONE) {
    __syncwarp();
    is = it;
    done = (int)first;
  } else {
    Item x;
    start = s_begin;
    set_sequence<ROWS, TILE>(p, x, s_b);
    while (first >= start + x.nt) { start += x.nt; next_item<ROWS, TILE>(p, x); }
    it = is = x;                                    // every lane writes the same
    done = (int)(first - start);
  }
  auto advance = [&](Item& s) {
    Item x = s;
    next_item<ROWS, TILE>(p, x);
    __syncwarp();
    s = x;
    __syncwarp();
  };

  // ---- ring: the issue side runs ST - 1 tiles ahead ----
  const uint32_t ring = su32(smem) + w * ST * SB, bar = su32(bars[w]);
  if (lane < ST) tc5::bar_init(&bars[w][lane], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  int to_issue = (int)(last - first), issued = 0, waited = 0;
  int is_left, is_slot, is_lo, is_hi, is_g, is_at = 0;     // tiles of the item not fetched yet, the warp's first token of the next
  // Pages of the item's next 32 tiles, a tile per lane, asked for while the tile before them is being computed: those of
  // the warp's first block and, where a page is one block, of its second.
  int pages[NB];
  auto look_up = [&]() {
    const int* table = c.table + (int64_t)is.b * c.W;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int first_slot = is_slot + lane * TILE + 16 * i, last_slot = first_slot + (c.shift == 4 ? 15 : STEP - 1);
      // only of what some row sees: below a window there may be no page
      const int j = first_slot >> c.shift;
      pages[i] = -1;
      if ((i == 0 || c.shift == 4) && first_slot < is_hi && last_slot >= is_lo && j < c.W) pages[i] = table[j];
    }
    is_at = 0;
  };
  auto fetch_item = [&](int skip) {
    is_left = is.nt - skip;
    is_slot = (is.k0 + skip) * TILE + w * STEP;
    is_lo = is.lo;
    is_hi = is.hi;
    is_g = is.g;
    look_up();
  };
  fetch_item(done);
  int flying = 0;                        // NB bits for each tile on its way, the next one's lowest: which blocks are there
  bool ok = true;
  auto issue = [&](uint32_t stage_at, uint32_t bar_at) {
    flying >>= NB;
    if (to_issue <= 0) return;
    ++issued;
    int pg[NB];
    pg[0] = __shfl_sync(0xffffffffu, pages[0], is_at);
#pragma unroll
    for (int i = 1; i < NB; ++i) pg[i] = c.shift == 4 ? __shfl_sync(0xffffffffu, pages[i], is_at) : pg[0];
    int there = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int slot = is_slot + 16 * i;
      const bool sees = slot < is_hi && slot + 16 > is_lo, page = (unsigned)pg[i] < (unsigned)c.P;
      there |= (sees && page) << i;
      bad = bad || (sees && !page);
    }
    flying |= there << NB * (ST - 1);
    if (lane == 0) {
      if (bad) record(ERR_PAGE);
      if (there)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar_at), "r"(__popc(there) * BLOCK<HD>) : "memory");
      else
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_at) : "memory");
      // blocks of one page are adjacent
      const bool whole = there == (1 << NB) - 1 && c.shift > 4;
      if (there & 1)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(stage_at), "l"(block_of<HD>(c, pg[0], is_g, is_slot)), "r"(whole ? SB : BLOCK<HD>), "r"(bar_at) : "memory");
      if (!whole) {
#pragma unroll
        for (int i = 1; i < NB; ++i)
          if (there >> i & 1)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(stage_at + i * BLOCK<HD>), "l"(block_of<HD>(c, pg[i], is_g, is_slot + 16 * i)), "r"(BLOCK<HD>), "r"(bar_at) : "memory");
      }
    }
    if (--to_issue > 0) {
      is_slot += TILE;
      ++is_at;
      if (--is_left == 0) {
        advance(is);
        fetch_item(0);
      } else if (is_at == 32) {
        look_up();
      }
    }
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(ring + s * SB, bar + s * 8);

  // ---- state of the current item ----
  uint32_t qf[NR][MT][2];
  float rs[NR][2];                        // score factor of rows 2 t4, 2 t4 + 1
  int it_hi = 0, all_lo = 0, all_hi = 0;             // slots [all_lo, all_hi] that every row sees
  float r[NR][2], l[NR][2], o[NR][MT][4]; // weights are 2^(score - r), at most 2^(LIFT + LAZY)
  float* scores_at = nullptr;             // of slot 0 and this lane's first row
  auto load_rows = [&]() {
    const int per = p.rep * p.maps, at0 = it.len - it.n;
    if (p.scores) {
      const int64_t at = it.rows <= p.stride ? scores_of(p, it.b, it.g) : NOT_KEPT;
      scores_at = at != NOT_KEPT ? p.scores + at * p.stride + 2 * t4 : nullptr;
    }
    it_hi = it.hi;
    all_hi = min(it.len - 1, at0 + it.rt * ROWS / per);
    all_lo = p.window > 0 ? at0 + min(it.n - 1, (it.rt * ROWS + ROWS - 1) / per) - p.window + 1 : 0;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int row = it.rt * ROWS + nr * 8 + g8;
      float f[KW][8];
      float mx = 0.f;
      if (row < it.rows) {
        const int i = row / per, h = it.g * p.rep + (row % per) / p.maps, map = row % p.maps;
        const T* q = map ? (const T*)p.q2 + (int64_t)(it.t0 + i) * p.st2 + (int64_t)h * p.sh2
                         : (const T*)p.q1 + (int64_t)(it.t0 + i) * p.st1 + (int64_t)h * p.sh1;
#pragma unroll
        for (int i2 = 0; i2 < KW / 2; ++i2) q_row16(q + t4 * (HD / 4) + 16 * i2, &f[2 * i2][0]);
#pragma unroll
        for (int i2 = 0; i2 < KW; ++i2)
#pragma unroll
          for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(f[i2][j]));
      } else {
#pragma unroll
        for (int i2 = 0; i2 < KW; ++i2)
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i2][j] = 0.f;
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^e <= mx < 2^(e + 1); rows of zeros and rows with infinities stay as they are
      int e = (int)(__float_as_uint(mx) >> 23) - 127;
      if (e == -127 || e == 128) e = 0;
      e = max(-126, min(126, e));
      // The factor of the scores is above 0: the largest product is the largest score, and what is masked stays so.  A
      // factor of 0, or one that underflows, gives scores of 0 all the same: products are below 2^25.
      const float down = __uint_as_float((uint32_t)(127 - e) << 23 | (p.scale_log2 < 0.f ? 0x80000000u : 0u)), up = __uint_as_float((uint32_t)(127 + e) << 23);
      // as the codes of a word are decoded: dims (0, 4) and (1, 5), then (2, 6) and (3, 7)
#pragma unroll
      for (int i2 = 0; i2 < KW; ++i2)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < 2; ++j) qf[nr][2 * i2 + y][j] = pack_h2(f[i2][2 * y + j] * down, f[i2][2 * y + j + 4] * down);
      const float mine_rs = fmaxf(fabsf(p.scale_log2) * up, 1e-37f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        rs[nr][x] = __shfl_sync(0xffffffffu, mine_rs, (2 * t4 + x) * 4);
        r[nr][x] = NONE;
        l[nr][x] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[nr][j][x] = 0.f;
    }
    __syncwarp();
    if (lane < ROWS) {
      // rows past the last one are rows of zeros that see everything: they ask for no mask and are not written
      const int row = it.rt * ROWS + lane, at = at0 + row / per;
      s_sees[w][lane] = row < it.rows ? make_int2(p.window > 0 ? at - p.window : -1, min(it.len - 1, at)) : make_int2(-1, 0x7fffffff);
    }
    __syncwarp();
  };

  // K rows of this lane in the fragments: tokens g8 and g8 + 8, dims HD / 4 t4 ..;  V: tokens 2 t4, 2 t4 + 1 and the same
  // + 8, dims HD / 8 g8 ..
  const uint32_t k_at = g8 * (HD / 2) + t4 * (HD / 8), kp_at = PARAMS<HD> + g8 * (HD / 16);
  const uint32_t v_at = HALF<HD> + 2 * t4 * (HD / 2) + g8 * (HD / 16), vp_at = HALF<HD> + PARAMS<HD> + 2 * t4 * (HD / 16);
  const Base base = c.base;
  // raw products of a block's keys
  auto products = [&](uint32_t kb, float (&s)[NR][4]) {
    uint32_t kw[2][KW];
    Levels lv[2][KW / 2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (HD == 128) {
        const uint4 v = lds16(kb + k_at + x * 8 * (HD / 2));
        const uint2 pw = lds8(kb + kp_at + x * 8 * (HD / 16));
        kw[x][0] = v.x; kw[x][1] = v.y; kw[x][KW - 2] = v.z; kw[x][KW - 1] = v.w;
        lv[x][0] = levels_of(pw.x, base); lv[x][KW / 2 - 1] = levels_of(pw.y, base);
      } else {
        const uint2 v = lds8(kb + k_at + x * 8 * (HD / 2));
        kw[x][0] = v.x; kw[x][1] = v.y;
        lv[x][0] = levels_of(lds4(kb + kp_at + x * 8 * (HD / 16)), base);
      }
    }
    // S^T: word i holds runs 2 i, 2 i + 1 of the lane's dims, of groups (0, 1) or (2, 3)
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      uint32_t a[4], b[4];
      decode(kw[0][i], lv[0][i % (KW / 2)], base, a);
      decode(kw[1][i], lv[1][i % (KW / 2)], base, b);
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        if (i == 0) mma_new(s[nr], a[0], b[0], a[1], b[1], qf[nr][0][0], qf[nr][0][1]);
        else mma(s[nr], a[0], b[0], a[1], b[1], qf[nr][2 * i][0], qf[nr][2 * i][1]);
        mma(s[nr], a[2], b[2], a[3], b[3], qf[nr][2 * i + 1][0], qf[nr][2 * i + 1][1]);
      }
    }
  };
  // raw products of the tile's blocks, -inf where a row does not see the token; times rs they are the scores (log2)
  auto scores = [&](uint32_t at, int slot0, int there, float (&s)[NB][NR][4]) {
#pragma unroll
    for (int i = 0; i < NB; ++i) products(at + i * BLOCK<HD>, s[i]);
    if (there != (1 << NB) - 1 || slot0 + STEP - 1 > all_hi || slot0 < all_lo) {
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int2 sees = s_sees[w][nr * 8 + 2 * t4 + y];
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int slot = slot0 + 16 * i + g8 + x * 8;
              if (slot > sees.y || slot <= sees.x || !(there >> i & 1)) s[i][nr][2 * x + y] = -INFINITY;
            }
        }
    }
    if (scores_at) {                              // rows 2 t4 and 2 t4 + 1 of tokens g8 and g8 + 8 of each block
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
        if (nr * 8 + 2 * t4 < p.stride) {
#pragma unroll
          for (int i = 0; i < NB; ++i)
            if (there >> i & 1) {
#pragma unroll
              for (int x = 0; x < 2; ++x)
                *reinterpret_cast<float2*>(scores_at + (int64_t)(slot0 + 16 * i + g8 + 8 * x) * p.stride + nr * 8) = make_float2(s[i][nr][2 * x] * rs[nr][0], s[i][nr][2 * x + 1] * rs[nr][1]);
            }
        }
    }
  };
  auto raise = [&](float (&s)[NB][NR][4]) {
    float mx[NR][2];
    bool grow = false;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[nr][x] = fmaxf(s[0][nr][x], s[0][nr][x + 2]);
#pragma unroll
        for (int i = 1; i < NB; ++i) mx[nr][x] = fmaxf(mx[nr][x], fmaxf(s[i][nr][x], s[i][nr][x + 2]));
        mx[nr][x] *= rs[nr][x];
        grow = grow || mx[nr][x] > r[nr][x] + (LIFT + LAZY);
      }
    if (!__any_sync(0xffffffffu, grow)) return;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float m = mx[nr][x];
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        const float r1 = fmaxf(r[nr][x], m - LIFT), f = ex2(r[nr][x] - r1);
        r[nr][x] = r1;
        l[nr][x] *= f;
#pragma unroll
        for (int j = 0; j < MT; ++j) { o[nr][j][x] *= f; o[nr][j][x + 2] *= f; }
      }
  };
  // P V of one block
  auto values = [&](uint32_t vb, int slot0, bool clear, float (&s)[NR][4]) {
    uint32_t pf[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        e[x] = ex2(fmaf(s[nr][x], rs[nr][x & 1], -r[nr][x & 1]));
        l[nr][x & 1] += e[x];
      }
      pf[nr][0] = transposed(pack_h2(e[0], e[1]));
      pf[nr][1] = transposed(pack_h2(e[2], e[3]));
    }
    // O^T: tokens 2 t4 (x = 0), 2 t4 + 1, and the same + 8 (x = 2, 3)
    uint32_t vw[4][VW], pw[4][VW];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = (x & 1) + (x >> 1) * 8;
      if (HD == 128) {
        const uint2 v = lds8(vb + v_at + row * (HD / 2)), u = lds8(vb + vp_at + row * (HD / 16));
        vw[x][0] = v.x; vw[x][VW - 1] = v.y;
        pw[x][0] = u.x; pw[x][VW - 1] = u.y;
      } else {
        vw[x][0] = lds4(vb + v_at + row * (HD / 2));
        pw[x][0] = lds4(vb + vp_at + row * (HD / 16));
      }
    }
    if (clear) {                                       // what is past the end, or not there, may be anything: zeros
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (slot0 + 2 * t4 + (x & 1) + (x >> 1) * 8 >= it_hi) {
#pragma unroll
          for (int i = 0; i < VW; ++i) pw[x][i] = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < VW; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // the word's lower and upper four dims, of one group each
        const uint32_t sel = h ? 0x7632u : 0x5410u;
        uint32_t a[4], b[4];
        decode(__byte_perm(vw[0][i], vw[1][i], sel), levels_of(__byte_perm(pw[0][i], pw[1][i], sel), base), base, a);
        decode(__byte_perm(vw[2][i], vw[3][i], sel), levels_of(__byte_perm(pw[2][i], pw[3][i], sel), base), base, b);
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          mma(o[nr][4 * i + 2 * h], a[0], a[1], b[0], b[1], pf[nr][0], pf[nr][1]);          // dims HD / 8 g8 + 8 i + 4 h, + 1
          mma(o[nr][4 * i + 2 * h + 1], a[2], a[3], b[2], b[3], pf[nr][0], pf[nr][1]);      // + 2, + 3
        }
      }
  };

  // Warps 3, 2, 1 pass their joined state on through shared memory, lane by lane; warp 0 writes the result.
  float* merge = reinterpret_cast<float*>(smem + NW * ST * SB) + lane;
  float* const s_part = reinterpret_cast<float*>(smem + NW * ST * SB + 32 * 4 * merge_words<HD, NR>());
  auto finish = [&](int64_t item_start, bool ends) {
#pragma unroll 1
    for (int turn = NW - 1; turn >= 0; --turn) {
      if (w == turn && turn < NW - 1) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float mm = merge[(nr * 4 + x) * 32], M = fmaxf(r[nr][x], mm);
            const float a = ex2(r[nr][x] - M), b = ex2(mm - M);
            r[nr][x] = M;
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
          for (int x = 0; x < 2; ++x) { merge[(nr * 4 + x) * 32] = r[nr][x]; merge[(nr * 4 + 2 + x) * 32] = l[nr][x]; }
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) merge[(NR * 4 + (nr * MT + j) * 4 + x) * 32] = o[nr][j][x];
        }
      }
      if (turn > 0) __syncthreads();
    }
    if (w == 0) {
      const bool whole = (!ALONE || gridDim.x == 1) && ends && item_start >= first, cut = *(volatile int*)&s_cut != 0;
      float* part = ALONE ? s_part : p.part + ((int64_t)blockIdx.x * 2 + (item_start > first ? 1 : 0)) * ROWS * (HD + 2);
      const int per = p.rep * p.maps;
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        float f0[2];                                     // 1 / sum over the row's lanes
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float M = r[nr][x];
          float L = l[nr][x];
          L += __shfl_xor_sync(0xffffffffu, L, 4);
          L += __shfl_xor_sync(0xffffffffu, L, 8);
          L += __shfl_xor_sync(0xffffffffu, L, 16);
          if (cut) L = -1.f;                             // in a part: the join writes zeros
          f0[x] = cut || L == 0.f ? 0.f : 1.f / L;
          const int part_row = nr * 8 + 2 * t4 + x;
          if (whole && p.lse && g8 == 0) {
            const int row = it.rt * ROWS + part_row;
            if (row < it.rows)
              p.lse[(int64_t)(it.t0 + row / per) * p.H * p.maps + it.g * per + row % per] = cut || L == 0.f ? INFINITY : M + log2f(L);
          }
          if (!whole) {
            float* dst = part + part_row * (HD + 2);
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
      if (!ALONE && ends && !whole && lane == 0) {
        const int64_t c0 = item_start / share;       // CTA and place of the item's first part
        p.joins[blockIdx.x] = make_int4(it.t0, it.rows, it.g | it.rt << 16, (int)(2 * c0 + (item_start > c0 * share ? 1 : 0)));
      }
    }
    __syncthreads();
  };

  load_rows();
  int tiles = it.nt - done;                                            // of the item, still to be done
  int slot0 = (it.k0 + done) * TILE + w * STEP;
  uint32_t here = ring, bar_here = bar, phase = 0, there = ring + (ST - 1) * SB, bar_there = bar + (ST - 1) * 8;
  if (ALONE && first == last) finish(start, true);   // no tile is left for this CTA: a part of nothing
  for (int left = (int)(last - first); left > 0; --left) {
    if (ok) {
      issue(there, bar_there);
      ok = wait_tile(bar_here, phase, p.wait);
      waited += ok;
      if (!ok) s_cut = 1;                          // this item's rows and the next ones' are zeros
    }
    const int blocks = flying & ((1 << NB) - 1);
    if (ok && blocks) {
      float s[NB][NR][4];
      scores(here, slot0, blocks, s);
      raise(s);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const bool not_there = !(blocks >> i & 1);
        values(here + i * BLOCK<HD>, not_there ? it_hi : slot0 + 16 * i, not_there || slot0 + 16 * (i + 1) > it_hi, s[i]);
      }
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
        advance(it);
        tiles = it.nt;
        slot0 = it.k0 * TILE + w * STEP;
        load_rows();
      }
    }
  }
  if (ALONE && gridDim.x > 1) {
    // the cluster's parts, a row (or a head's pair of rows) per CTA and turn, 32 dims a warp
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int C = gridDim.x, per = p.rep * p.maps, n_rows = min(ROWS, it.rows - it.rt * ROWS);
    for (int rr = rank * p.maps; rr < n_rows; rr += C * p.maps) {
      const int row = it.rt * ROWS + rr, tok = it.t0 + row / per, h = it.g * p.rep + row % per / p.maps;
      for (int d = tid; d < HD; d += NT) {
        float x[2] = {0.f, 0.f};
        bool cut = false;
        for (int map = 0; map < p.maps; ++map) {
          const float* src = s_part + (rr + map) * (HD + 2);
          float2 ml[MOST];
          float v[MOST];
#pragma unroll
          for (int i = 0; i < MOST; ++i) {
            ml[i] = make_float2(NONE, 0.f);
            v[i] = 0.f;
            if (i < C) {
              const float* remote = cluster.map_shared_rank(src, i);
              ml[i] = *reinterpret_cast<const float2*>(remote + HD);
              v[i] = remote[d];
            }
          }
          float M = NONE, L = 0.f, a = 0.f;
#pragma unroll
          for (int i = 0; i < MOST; ++i) M = fmaxf(M, ml[i].x);
#pragma unroll
          for (int i = 0; i < MOST; ++i) {
            const float e = ex2(ml[i].x - M);
            cut = cut || ml[i].y < 0.f;
            L = fmaf(ml[i].y, e, L);
            a = fmaf(v[i], e, a);
          }
          x[map] = L == 0.f ? 0.f : a / L;
          if (p.lse && d == 0) p.lse[(int64_t)tok * p.H * p.maps + it.g * per + row % per + map] = L == 0.f ? INFINITY : M + log2f(L);
        }
        if (p.maps == 2) x[0] = (x[0] - p.lam[h] * x[1]) / (1.f - p.lam[h] + 1e-8f);
        if (cut && p.lse && d == 0)
          for (int map = 0; map < p.maps; ++map) p.lse[(int64_t)tok * p.H * p.maps + it.g * per + row % per + map] = INFINITY;
        ((T*)p.out)[((int64_t)tok * p.H + h) * HD + d] = from_f<T>(cut ? 0.f : x[0]);
      }
    }
    cluster.sync();                                 // nobody leaves while its part is read
  }
  // after a wait that ran out: the copies that are still under way into this CTA's memory
  for (; waited < issued; ++waited) drain_tile(bar + waited % ST * 8, (uint32_t)(waited / ST & 1));
}

// ---- received weights ------------------------------------------------------------------------------
// Where each sequence's scores go when the workspace is as large as the pool: one block lays the pages that rows see end to
// end.  They are one sequence's each, so they fit; what does not is recorded and left out.
constexpr int NPL = 1024;
__global__ void __launch_bounds__(NPL) places_kernel(const __grid_constant__ Params p, Place* places, int64_t room) {
  const Cache4& c = p.c;
  const int chunk = (c.B + NPL - 1) / NPL, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto place_of = [&](int b) {
    Item it;
    Place at{-1, 0, 0};
    if (!in_order(c, b) || !set_sequence<2 * 8, TILE>(p, it, b) || it.rows > p.stride) return at;
    at.start = 0;
    at.lo = it.lo >> c.shift << c.shift;
    at.n = max(0, ((it.hi + c.page - 1) >> c.shift << c.shift) - at.lo);
    return at;
  };
  const int b0 = threadIdx.x * chunk, b1 = min(c.B, b0 + chunk);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += place_of(b).n;
  __shared__ int64_t sums[NPL / 32];
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sums[w] = incl;
  __syncthreads();
  for (int i = 0; i < w; ++i) incl += sums[i];
  int64_t at = incl - mine;
  for (int b = b0; b < b1; ++b) {
    Place x = place_of(b);
    if (x.start == 0) {
      x.start = at;
      at += x.n;
      if (at > room) { x.start = -1; record(ERR_PAGE); }
    }
    places[b] = x;
  }
}

// From the scores that the split kernel has left: a thread per slot.
constexpr int NK = 256;
// all of an SM's threads resident: 32 registers; with 35, 64 sequences of up to 8191 slots took 20 us and not 17
__global__ void __launch_bounds__(NK, 8) kept_weights_kernel(const __grid_constant__ Params p) {
  const Cache4& c = p.c;
  const int g = blockIdx.y, b = blockIdx.z;
  Item it;
  if (!in_order(c, b) || !set_sequence<2 * 8, TILE>(p, it, b) || it.rows > p.stride) return;
  const int64_t first = scores_of(p, b, g);
  if (first == NOT_KEPT) return;
  const int per = p.rep * p.maps;
  __shared__ float lse[KEEP];
  if (threadIdx.x < KEEP) {
    const int row = threadIdx.x;
    lse[row] = row < it.rows ? p.lse[(int64_t)(it.t0 + row / per) * p.H * p.maps + g * per + row % per] : INFINITY;
  }
  __syncthreads();
  // rows cut short (+inf) have not left all of their scores
  auto weight = [](float score, float of) { return of == INFINITY ? 0.f : ex2(score - of); };
  for (int slot = it.lo / 16 * 16 + blockIdx.x * NK + threadIdx.x; slot < it.hi; slot += gridDim.x * NK) {
    const int pg = c.table[(int64_t)b * c.W + (slot >> c.shift)];
    if (pg < 0 || pg >= c.P) continue;                  // recorded where its keys were looked for
    float* to = c.mass + (((int64_t)pg * c.G + g) << c.shift) + (slot & (c.page - 1));
    const float had = *to;
    const float* s = p.scores + (first + slot) * p.stride;
    float sum = 0.f;
    if (p.stride % 4 == 0) {
      for (int row = 0; row < it.rows; row += 4) {
        const float4 v = *reinterpret_cast<const float4*>(s + row);
        sum += (weight(v.x, lse[row]) + weight(v.y, lse[row + 1])) + (weight(v.z, lse[row + 2]) + weight(v.w, lse[row + 3]));
      }
    } else {
      for (int row = 0; row < it.rows; row += 2) {
        const float2 v = *reinterpret_cast<const float2*>(s + row);
        sum += weight(v.x, lse[row]) + weight(v.y, lse[row + 1]);
      }
    }
    *to = had + sum;
  }
}

template <typename T, int HD, int NR, bool ALONE>
void launch_split(const Params& p, int row_tiles, int cluster) {
  auto fn = split_kernel<T, HD, NR, ALONE>;
  constexpr int SMEM = smem_bytes<HD, NR, ALONE>();
  static bool set[64] = {};                              // by device; the attribute stays
  int dev = 0;
  MAMF_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 64 || !set[dev]) {
    MAMF_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) set[dev] = true;
  }
  if (!ALONE) {
    fn<<<p.ctas, NT, SMEM, stream()>>>(p);
    MAMF_LAUNCH_CHECK();
    launch_join<T, HD, NR>(p);
    return;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)cluster, (unsigned)(p.c.G * row_tiles), (unsigned)p.c.B);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fn, p));
}
template <typename T, int HD, int NR>
void launch_split(const Params& p, int row_tiles, int cluster) {
  if (cluster) launch_split<T, HD, NR, true>(p, row_tiles, cluster); else launch_split<T, HD, NR, false>(p, 0, 0);
}

}  // namespace pa4

// q1, q2 (T, H, hd) bf16 or f16 packed queries -> (T, H, hd)
at::Tensor paged4_attention(at::Tensor q1, c10::optional<at::Tensor> q2, c10::optional<at::Tensor> lam, at::Tensor blocks,
                            c10::optional<at::Tensor> mass, at::Tensor table, at::Tensor cu, at::Tensor lens,
                            int64_t max_new, int64_t window, double scale) {
  using namespace pa4;
  TORCH_CHECK(q1.is_cuda() && q1.dim() == 3 && q1.device() == blocks.device() && (q1.scalar_type() == at::kBFloat16 || q1.scalar_type() == at::kHalf),
              "paged_attention: bf16 or f16 queries (T, H, hd) on the cache's GPU");
  c10::cuda::CUDAGuard guard(q1.device());
  const int64_t T = q1.size(0), H = q1.size(1), hd = q1.size(2);
  Params p{};
  p.c = check_cache4("paged_attention", blocks, mass, table, &cu, lens, T, hd);
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
  p.wait = attention_wait_limit();
  p.rep = (int)(H / p.c.G);
  p.maps = p.q2 ? 2 : 1;
  p.cap = (int64_t)p.c.W * p.c.page;
  TORCH_CHECK(T * H < (1LL << 31), "paged_attention: sizes");
  // Sequences of up to FEW rows go to the split kernel, longer runs of tokens to the chunk kernel; where all
  // have the same number of tokens one of them does everything.
  const int64_t most_rows = std::max<int64_t>(1, std::min(max_new, T)) * p.rep * p.maps;
  p.chunked = most_rows > FEW && p.c.B > 0;
  const bool alone = p.chunked && T == p.c.B * max_new;
  p.few = alone ? 0 : (int)std::min<int64_t>(most_rows, FEW);
  at::Tensor sums, kept, places;
  if (mass.has_value() && p.c.B > 0) {
    TORCH_CHECK(p.c.B < 65536, "paged_attention: received weights of at most 65535 sequences");
    sums = at::empty({T, H, p.maps}, q1.options().dtype(at::kFloat));
    p.lse = sums.data_ptr<float>();
    if (!alone) {
      p.stride = (int)((std::min<int64_t>(p.few, KEEP) + 1) / 2 * 2);
      // A place for each slot that the block table has room for, or, where that is far more than the pool has, for each
      // of the pool's: one launch more.
      const int64_t pool = (int64_t)p.c.P * p.c.page, room = p.c.B * p.cap;
      const bool dense = 2 * pool < room;
      kept = at::empty({(dense ? pool : room) * p.c.G * p.stride}, q1.options().dtype(at::kFloat));
      p.scores = kept.data_ptr<float>();
      if (dense) {
        places = at::empty({(int64_t)p.c.B * (int64_t)sizeof(Place)}, q1.options().dtype(at::kByte));
        Place* to = reinterpret_cast<Place*>(places.data_ptr<uint8_t>());
        p.places = to;
        places_kernel<<<1, NPL, 0, stream()>>>(p, to, pool);
        MAMF_LAUNCH_CHECK();
      }
    }
  }
  const bool bf16 = q1.scalar_type() == at::kBFloat16;
  if (p.chunked) chunk_attention(p, (int)hd, bf16);
  if (!alone) {
    // one query row tile holds 8 rows, or 16 where a sequence can have more than 8
    const int nr = p.few > 8 ? 2 : 1, rows = 8 * nr;
    const int64_t row_tiles = (p.few + rows - 1) / rows;
    const int64_t tiles = std::max<int64_t>(1, (p.cap + TILE - 1) / TILE);
    int cluster = 0;
    at::Tensor ws;
    const int64_t slots = (nr == 1 ? residents<128, 1>() : hd == 64 ? residents<64, 2>() : residents<128, 2>()) * num_sms();
    const int64_t items = (int64_t)p.c.B * p.c.G * row_tiles;
    if (items > 0 && !p.chunked) {
      cluster = MOST;
      while (cluster > 1 && (items * cluster > slots || cluster >= 2 * tiles)) cluster /= 2;
      if (items * cluster > slots || tiles > SHORT * cluster) cluster = 0;
    }
    if (!cluster) {
      const int64_t most = std::max<int64_t>(1, items * tiles);
      p.ctas = (int)std::min<int64_t>(most, slots);
      const int64_t part = (int64_t)p.ctas * 2 * rows * (hd + 2);
      ws = at::empty({part + 4 * p.ctas}, q1.options().dtype(at::kFloat));
      p.joins = reinterpret_cast<int4*>(ws.data_ptr<float>());
      p.part = ws.data_ptr<float>() + 4 * p.ctas;
    }
    auto go = [&](auto t) {
      using E = decltype(t);
      if (hd == 128) { if (nr == 1) launch_split<E, 128, 1>(p, (int)row_tiles, cluster); else launch_split<E, 128, 2>(p, (int)row_tiles, cluster); }
      else { if (nr == 1) launch_split<E, 64, 1>(p, (int)row_tiles, cluster); else launch_split<E, 64, 2>(p, (int)row_tiles, cluster); }
    };
    if (bf16) go(__nv_bfloat16()); else go(__half());
  }
  if (p.lse) {
    if (p.scores) {
      kept_weights_kernel<<<dim3((unsigned)((p.cap + 4 * NK - 1) / (4 * NK)), (unsigned)p.c.G, (unsigned)p.c.B), NK, 0, stream()>>>(p);
      MAMF_LAUNCH_CHECK();
    }
    if (most_rows > p.stride) chunk_weights(p, p.stride, (int)hd, bf16);
  }
  return out;
}

int64_t paged4_attention_error(bool clear) {
  return paged::take_code(split::g_err, clear) | paged::take_code(split::g_wait_err, clear) | paged4::chunk_error(clear);
}

}  // namespace mamf
