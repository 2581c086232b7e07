// Attention over the paged 4-bit cache (layout in paged4.cuh) for many query rows per KV head: chunks of a prompt.  The
// products run on the 5th-generation tensor cores; every key tile is read once per CTA.
//
// A CTA holds two streams of 128 query rows of one KV head that share its keys and values:
//   differential: the two maps of the same rows;   single softmax: two neighbouring tiles of rows.
// A row is (token, head of the group), so short runs of tokens still fill a tile.  11 warps:
//   warps 0-3, 4-7  softmax of stream A, B (thread = row = TMEM lane): write the row of q to shared memory
//                   as f16, scaled by a power of two to [1, 2); then S from TMEM, P as packed f16 back over it
//   warps 8-9       keys and values: 64-token tiles, 16 bytes of codes per load, through registers one tile ahead,
//                   decoded to f16 (exact) into a ring of 128-byte-swizzled tiles; tokens past the end become 0
//   warp 10         TMEM allocation, MMA issue: S = Q K^T (M 128, N 64), O += P V (N = head size, P in TMEM)
// Where there are fewer tiles than SMs, several CTAs share a tile's keys and a second kernel joins them.  Online softmax
// with lazy rescaling as in flash_tc.cu.  Every wait is bounded; a wait that runs out records a code, and the CTA winds
// down and leaves zeros.
//
// P is rounded to f16 (11 bits of a weight) at up to 2^15, so that weights down to 2^-21 of a row's largest keep them; its
// sum is fp32.
//
// 4 x 1024 tokens on 7168 cached, 32 / 8 heads of 128: two maps 1.37 ms, 752 TFLOP/s, one 0.78 ms, 665 TFLOP/s.  Bound by the
// hand-offs of the 64-key tiles between its roles, as the 8-bit kernel of the same shape (1.22 ms, 0.68): tensor pipe 35%,
// exponentials 36%, 39% of the issue slots.  Decoding 4 bits takes the two converting warps more instructions than e4m3 does.
#include "f32x2.cuh"
#include "paged4.cuh"
#include "tc5.cuh"

namespace mamf {
namespace ptc4 {

using namespace paged4;
using namespace tc5;

constexpr int BM = 128, BN = 64, ST = 4, NC = 64, NT = 256 + NC + 32;       // NC converting threads
constexpr float LIFT = 7.f, LAZY = 8.f, NONE = -1e30f;      // as in the split kernel

__device__ int g_err = 0, g_wait_err = 0;

template <int HD> constexpr int q_bytes() { return BM * HD * 2; }
template <int HD> constexpr int k_bytes() { return BN * HD * 2; }
// the epilogue's exchange rows (fp32) lie over Q and the ring
template <int HD> constexpr int smem_bytes() { return 1024 + 2 * q_bytes<HD>() + 2 * ST * k_bytes<HD>(); }

struct Params : Attn4 {
  int splits;          // CTAs that share a tile's keys; with more than one they leave parts for the join kernel:
  float* part;         // [unit * G + head][split][stream][BM][HD + 2]: O (not divided), m, l
};

// As tc5::bar_wait, without its suspend-time hint: the hand-offs of a tile are short (on the 8-bit kernel, 1.72 ms against
// 1.77).  The error
// word is only written here: a wait that ran out in another CTA, or in an earlier call, ends no wait of this one.  After
// one that ran out a role waits for nothing more, so a CTA ends within a few limits.
__device__ __forceinline__ bool try_once(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok) : "r"(su32(b)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint64_t* b, uint32_t parity, long long limit) {
  if (limit >= 0 && try_once(b, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t n = 1;; ++n) {
    if (limit >= 0 && try_once(b, parity)) return true;
    if ((n & 1023u) == 0 && clock64() - t0 > limit) {
      atomicCAS(&g_wait_err, 0, (int)ERR_WAIT);
      return false;
    }
  }
}
// kind::f16, f16 x f16 -> fp32, A K-major
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ uint32_t h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The column of O, of 8, that holds dim d: the converting threads lay dims out as their codes are decoded.
__host__ __device__ constexpr int place(int d) { return (d & ~7) + 2 * (d & 3) + (d >> 2 & 1); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T, int HD>
__global__ void __launch_bounds__(NT, 1) chunk_kernel(const __grid_constant__ Params p) {
  constexpr int QB = q_bytes<HD>(), KB = k_bytes<HD>();
  constexpr int O_COL = 256;                       // TMEM: S_A[2], S_B[2] of 64 columns, then O_A, O_B of HD
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t q_full, kv_full[ST], kv_empty[ST], s_full[4], p_full[4], o_done[4], ex_full, idle;
  __shared__ int groups[ST];                       // bit q: the q-th block of a tile is there
  __shared__ uint32_t tmem_slot;
  __shared__ int cut;                              // a wait of the second map ran out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cache4& c = p.c;

  if (p.few == 0 && blockIdx.y == 0) {             // no other kernel runs: rows before the first and past the last sequence
    const int64_t row = (int64_t)p.H * HD, first = min(max(0, c.cu[0]), c.T) * row, end = max(0, c.cu[c.B]) * row;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < first; i += (int64_t)gridDim.x * NT) ((T*)p.out)[i] = from_f<T>(0.f);
    for (int64_t i = end + (int64_t)blockIdx.x * NT + threadIdx.x; i < c.T * row; i += (int64_t)gridDim.x * NT)
      ((T*)p.out)[i] = from_f<T>(0.f);
    if (blockIdx.x == gridDim.x - 1) {             // one CTA, of rows that see little, looks at all offsets
      bool odd = false;
      bool long_one = false;
      for (int i = threadIdx.x; i < c.B; i += NT) {
        odd = odd || !in_order(c, i);
        long_one = long_one || cached_length(c, c.lens[i]) != c.lens[i];
      }
      if (long_one || odd) atomicCAS(&g_err, 0, (int)ERR_LENGTH);
      if (__syncthreads_or(odd)) {                 // none of the call's results count, and nobody else writes any
        for (int64_t i = threadIdx.x; i < c.T * row; i += NT) ((T*)p.out)[i] = from_f<T>(0.f);
        if (p.lse)
          for (int64_t i = threadIdx.x; i < (int64_t)c.T * p.H * p.maps; i += NT) p.lse[i] = INFINITY;
      }
    }
  }
  // ---- the CTA's rows ----
  const int rows = p.maps == 2 ? BM : 2 * BM;      // (token, head) pairs per CTA
  const int g = blockIdx.x % c.G;
  const int u = (gridDim.x - 1 - blockIdx.x) / c.G;        // later rows, which see more, first
  // unit numbers of sequence b start at cu[b] rep / rows + b: it has ceil(n rep / rows) tiles or less
  int b = 0;
  {
    int hi = c.B - 1;
    while (b < hi) {
      const int mid = (b + hi + 1) >> 1;
      if ((int64_t)c.cu[mid] * p.rep / rows + mid <= u) b = mid; else hi = mid - 1;
    }
  }
  const int t0 = c.cu[b], n = c.cu[b + 1] - t0, len = cached_length(c, c.lens[b]);
  const int64_t tile64 = u - ((int64_t)t0 * p.rep / rows + b);
  if (!in_order(c, b) || (int64_t)n * p.rep * p.maps <= p.few || tile64 < 0 || tile64 * rows >= (int64_t)n * p.rep) return;
  const int r0 = (int)tile64 * rows, total = n * p.rep;    // first row of the tile, rows of the sequence
  const int at0 = len - n;                                 // slot of token 0
  const int i0 = r0 / p.rep, i1 = min(n - 1, (r0 + rows - 1) / p.rep);
  const int key_hi = max(0, min(len, at0 + i1 + 1));
  const int key_lo = p.window > 0 ? max(0, at0 + i0 - p.window + 1) : 0;
  int kt0 = key_lo / BN;
  int ntile = key_hi > key_lo ? (key_hi + BN - 1) / BN - kt0 : 0;
  if (p.splits > 1) {                              // this CTA's share of the key tiles
    const int share = (ntile + p.splits - 1) / p.splits, first = min(ntile, (int)blockIdx.y * share);
    kt0 += first;
    ntile = min(share, ntile - first);
  }

  // Offsets out of order anywhere: some rows may be no unit's, or two units', so no unit leaves results.  The look at them is
  // over by the time that the tensor memory is there.
  bool odd = false;
  for (int i = threadIdx.x; i < c.B; i += NT) odd = odd || !in_order(c, i);
  if (threadIdx.x == 0) {
    bar_init(&q_full, 256);
    bar_init(&ex_full, 128);
    bar_init(&idle, 1);
    cut = 0;
    for (int s = 0; s < ST; ++s) { bar_init(&kv_full[s], NC / 32); bar_init(&kv_empty[s], 1); }
    for (int i = 0; i < 4; ++i) { bar_init(&s_full[i], 1); bar_init(&p_full[i], 128); bar_init(&o_done[i], 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8 + NC / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  odd = __syncthreads_or(odd);
  fence_after();
  const uint32_t tmem = tmem_slot;
  if (odd) {
    if (warp == 8 + NC / 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    return;
  }
  uint8_t* ring = sm + 2 * QB;

  if (warp >= 8 && warp < 8 + NC / 32) {
    // ------------------------------- keys and values -------------------------------
    // A thread converts N chunks of 16 bytes of codes (32 dims) of keys and of values, RS tokens apart.
    constexpr int CR = HD / 32, N = BN * CR / NC, RS = NC / CR;
    const int ct = threadIdx.x - 256, r0c = ct / CR, cc = ct % CR;
    uint4 kx[N], vx[N];                                      // chunk i: token i RS + r0c, dims 32 cc ..
    uint32_t kp[N][HD / 64], vp[N][HD / 64];                 // the token's parameters
    int there = 0;                                           // bit q: block q of the tile is there
    auto look_up = [&](int j) {                              // the page of block lane % 4 of tile j
      const int slot = (kt0 + j) * BN + (lane & 3) * 16;
      if (j >= ntile || slot >= key_hi || slot + 16 <= key_lo) return -2;      // nothing to see there: no page is asked for
      const int w = slot >> c.shift;
      const int pg = w < c.W ? c.table[(int64_t)b * c.W + w] : -1;
      return (unsigned)pg < (unsigned)c.P ? pg : -1;
    };
    auto load = [&](int j, int pg) {
      const int slot = (kt0 + j) * BN;
      if (pg == -1 && ct < 4) atomicCAS(&g_err, 0, (int)ERR_PAGE);
      there = (int)__ballot_sync(0xffffffffu, pg >= 0) & 15;
      const int64_t mine = pg >= 0 ? block_of<HD>(c, pg, g, slot + (lane & 3) * 16) - c.blocks : -1;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int tok = i * RS + r0c;                        // its block is the same for a warp where RS is 16
        const int64_t off = __shfl_sync(0xffffffffu, mine, tok >> 4);
        kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) kp[i][x] = vp[i][x] = 0;         // what stands for zeros, whatever the codes
        if (off >= 0 && slot + tok < key_hi) {               // what is past the end may be anything
          const uint8_t* blk = c.blocks + off;
          kx[i] = *reinterpret_cast<const uint4*>(blk + (tok & 15) * (HD / 2) + cc * 16);
          vx[i] = *reinterpret_cast<const uint4*>(blk + HALF<HD> + (tok & 15) * (HD / 2) + cc * 16);
          const uint32_t* pk = reinterpret_cast<const uint32_t*>(blk + PARAMS<HD> + (tok & 15) * (HD / 16));
#pragma unroll
          for (int x = 0; x < HD / 64; ++x) { kp[i][x] = pk[x]; vp[i][x] = pk[HALF<HD> / 4 + x]; }
        }
      }
    };
    // A word's 8 dims become 16 bytes, in the order (0, 4, 1, 5, 2, 6, 3, 7): the queries are laid out alike, and the rows
    // of O are put back in order when they are written.  The lanes of the second 64 dims store their words two places
    // further round: the banks of both differ.
    uint8_t* const at = ring + (cc >> 1) * (BN * 128) + r0c * 128;
    const int c0 = HD == 128 ? (cc & 1) * 4 : cc * 4, turn = HD == 128 ? cc & 2 : 0;
    const Base base = c.base;
    auto store = [&](uint8_t* row, const uint4& x, const uint32_t (&params)[HD / 64]) {
      Levels lv[HD / 64];
#pragma unroll
      for (int i = 0; i < HD / 64; ++i) lv[i] = levels_of(params[i], base);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int m = 0; m < 4; ++m) {                          // words m and m + 2 are of the same groups
        uint32_t h[4];
        decode(turn ? w[m ^ 2] : w[m], lv[HD == 128 ? m & 1 : 0], base, h);
        *reinterpret_cast<uint4*>(row + (((c0 + (m ^ turn)) ^ (r0c & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    };
    if (ntile > 0) load(0, look_up(0));
    int next = look_up(1);
    bool ok = true;
    for (int j = 0; j < ntile; ++j) {
      const int st = j % ST;
      if (j >= ST) ok = __all_sync(0xffffffffu, wait(&kv_empty[st], (uint32_t)((j / ST - 1) & 1), p.wait));
      if (!ok) break;
      if (ct == 0) groups[st] = there;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        store(at + st * 2 * KB + i * RS * 128, kx[i], kp[i]);
        store(at + st * 2 * KB + KB + i * RS * 128, vx[i], vp[i]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) bar_arrive(&kv_full[st]);
      if (j + 1 < ntile) {
        const int pg = next;
        next = look_up(j + 2);
        load(j + 1, pg);
      }
    }
  } else if (warp == 8 + NC / 32) {
    // ------------------------------- MMA issue -------------------------------
    if (lane == 0 && ntile > 0) {
      bool ok = wait(&q_full, 0, p.wait);
      fence_after();
      constexpr uint32_t ID_QK = idesc(BN, false), ID_PV = idesc(HD, true);
      auto issue_qk = [&](int j) -> bool {
        const int st = j % ST, buf = j & 1;
        // the S buffer last held P(j - 2), read by the O += P V that this thread issued before
        if (!wait(&kv_full[st], (uint32_t)((j / ST) & 1), p.wait)) return false;
        fence_after();
        const uint32_t kb = su32(ring + st * 2 * KB);
        for (int s = 0; s < 2; ++s) {
          const uint32_t qb = su32(sm + s * QB);
          const uint32_t d = tmem + (uint32_t)(s * 128 + buf * 64);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            mma_ss(d, sdesc(qb + (k >> 2) * (BM * 128) + (k & 3) * 32, 16, 1024), sdesc(kb + (k >> 2) * (BN * 128) + (k & 3) * 32, 16, 1024),
                   ID_QK, k > 0 ? 1u : 0u);
          commit(&s_full[s * 2 + buf]);
        }
        return true;
      };
      if (ok) ok = issue_qk(0);
      for (int j = 0; j < ntile && ok; ++j) {
        if (j + 1 < ntile && !issue_qk(j + 1)) { ok = false; break; }
        const int st = j % ST, buf = j & 1;
        const uint32_t vb = su32(ring + st * 2 * KB + KB);
        for (int s = 0; s < 2 && ok; ++s) {
          if (!wait(&p_full[s * 2 + buf], (uint32_t)((j >> 1) & 1), p.wait)) { ok = false; break; }
          fence_after();
          const uint32_t pa = tmem + (uint32_t)(s * 128 + buf * 64);
          const uint32_t d = tmem + (uint32_t)(O_COL + s * HD);
#pragma unroll
          for (int k = 0; k < BN / 16; ++k)
            mma_ts(d, pa + (uint32_t)(k * 8), sdesc(vb + k * 2048, BN * 128, 1024), ID_PV, (j > 0 || k > 0) ? 1u : 0u);
          commit(&o_done[s * 2 + buf]);
        }
        if (ok) commit(&kv_empty[st]);
      }
      // products under way read shared memory and write TMEM, both of which go when the CTA ends: where a wait has run
      // out, nobody else waits for them
      commit(&idle);
      for (const long long t = clock64(); !try_once(&idle, 0) && clock64() - t <= WAIT_CYCLES;) {}
    }
  } else if (warp < 8) {
    // ------------------------------- softmax -------------------------------
    const int s = warp >> 2, r = (warp & 3) * 32 + lane;    // stream, row in its tile = TMEM lane
    const int row = r0 + r + (p.maps == 1 ? s * BM : 0);
    const bool row_ok = row < total;
    const int i = row / p.rep, h = g * p.rep + row % p.rep;
    const int at = at0 + i;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float rs = 0.f;
    {
      const bool second = p.maps == 2 && s == 1;
      const T* q = second ? (const T*)p.q2 + (int64_t)(t0 + i) * p.st2 + (int64_t)h * p.sh2
                          : (const T*)p.q1 + (int64_t)(t0 + i) * p.st1 + (int64_t)h * p.sh1;
      Vec16<T> x[HD / 8];
      float mx = 0.f;
#pragma unroll
      for (int k = 0; k < HD / 8; ++k) {
        x[k].raw = make_uint4(0, 0, 0, 0);
        if (row_ok) x[k] = ld16(q + 8 * k);
      }
#pragma unroll
      for (int k = 0; k < HD / 8; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(to_f(x[k].v[j])));
      int e = (int)(__float_as_uint(mx) >> 23) - 127;       // rows of zeros and rows with infinities stay as they are
      if (e == -127 || e == 128) e = 0;
      e = max(-126, min(126, e));
      // the factor of the scores is not negative, so that the largest product is the largest score: its sign is q's
      const float down = p.scale_log2 < 0.f ? -pow2(-e) : pow2(-e);
      rs = fabsf(p.scale_log2) * pow2(e);
      uint8_t* qrow = sm + s * QB + r * 128;
#pragma unroll
      for (int k = 0; k < HD / 8; ++k) {
        uint4 v;
        v.x = h2(to_f(x[k].v[0]) * down, to_f(x[k].v[4]) * down);
        v.y = h2(to_f(x[k].v[1]) * down, to_f(x[k].v[5]) * down);
        v.z = h2(to_f(x[k].v[2]) * down, to_f(x[k].v[6]) * down);
        v.w = h2(to_f(x[k].v[3]) * down, to_f(x[k].v[7]) * down);
        *reinterpret_cast<uint4*>(qrow + (k >> 3) * (BM * 128) + (((k & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_async_smem();
      bar_arrive(&q_full);
    }
    // slots [lo, hi] that the row sees; rows past the last one (zeros) see everything and are not written
    const int hi = row_ok ? min(len - 1, at) : 0x7fffffff, lo = row_ok && p.window > 0 ? at - p.window + 1 : 0;
    float m = NONE, l = 0.f;                                 // weights are 2^(score - m), at most 2^(LIFT + LAZY)
    bool ok = true;
    for (int j = 0; j < ntile && ok; ++j) {
      const int buf = j & 1, st = j % ST;
      ok = __all_sync(0xffffffffu, wait(&kv_full[st], (uint32_t)((j / ST) & 1), p.wait) && wait(&s_full[s * 2 + buf], (uint32_t)((j >> 1) & 1), p.wait));
      if (!ok) break;
      fence_after();
      float sv[BN];
      tld64(tl + (uint32_t)(s * 128 + buf * 64), sv);
      const int gr = groups[st];
      float f = rs;
      const int kbase = (kt0 + j) * BN;
      if (__any_sync(0xffffffffu, !(gr == 15 && kbase >= lo && kbase + BN - 1 <= hi))) {
#pragma unroll
        for (int k = 0; k < BN; ++k) {
          const int key = kbase + k;
          sv[k] = (key >= lo && key <= hi && (gr >> (k >> 4) & 1)) ? sv[k] : -INFINITY;
        }
        // a factor that is 0, or underflows, would make a masked score's -inf NaN; products are below 2^25, so that this
        // one's scores are 0 all the same
        f = fmaxf(rs, 1e-37f);
      }
      float mq[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) mq[k] = fmaxf(fmaxf(sv[k], sv[8 + k]), fmaxf(sv[16 + k], sv[24 + k]));
#pragma unroll
      for (int k = 0; k < 8; ++k) mq[k] = fmaxf(fmaxf(fmaxf(mq[k], sv[32 + k]), fmaxf(sv[40 + k], sv[48 + k])), sv[56 + k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) mq[k] = fmaxf(mq[k], mq[k + 4]);
      const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * f;
      float fo = 1.f;
      if (mx > m + (LIFT + LAZY)) {
        const float m1 = mx - LIFT;
        fo = ex2(m - m1);                                   // 0 for the first key of a row
        l *= fo;
        m = m1;
      }
      if (j > 0 && __any_sync(0xffffffffu, fo != 1.f)) {
        ok = __all_sync(0xffffffffu, wait(&o_done[s * 2 + ((j - 1) & 1)], (uint32_t)(((j - 1) >> 1) & 1), p.wait));
        if (!ok) break;
        fence_after();
#pragma unroll 1
        for (int cc = 0; cc < HD; cc += 32) {
          float o[32];
          tld32(tl + (uint32_t)(O_COL + s * HD + cc), o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] *= fo;
          tst32(tl + (uint32_t)(O_COL + s * HD + cc), o);
        }
      }
      float pk_[BN / 2];                                    // P as f16 pairs, bit patterns in fp32 registers
      const uint64_t ff = pk(f, f), nn = pk(-m, -m);
      uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int q = 0; q < BN / 2; ++q) {
        float e0, e1;
        unpk(fma2(pk(sv[2 * q], sv[2 * q + 1]), ff, nn), e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        sum[q & 3] = add2(sum[q & 3], pk(e0, e1));
        pk_[q] = __uint_as_float(h2(e0, e1));
      }
      float s0, s1;
      unpk(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
      l += s0 + s1;
      tst32(tl + (uint32_t)(s * 128 + buf * 64), pk_);      // over this row's S, which is in registers
      fence_before();
      bar_arrive(&p_full[s * 2 + buf]);
    }
    // ---- result ----
    if (ok && ntile > 0) {
      ok = __all_sync(0xffffffffu, wait(&o_done[s * 2 + ((ntile - 1) & 1)], (uint32_t)(((ntile - 1) >> 1) & 1), p.wait));
      fence_after();
    }
    T* out = (T*)p.out + ((int64_t)(t0 + i) * p.H + h) * HD;
    if (p.splits == 1) {
      // Rows of zeros: no row sees a key, and then there is no wait for O either, which orders the exchange below after
      // the stores of q; or a wait has run out, in this warp or in the other map's.
      bool zeros = !ok || ntile == 0;
      if (p.maps == 2 && s == 1 && !ok) cut = 1;
      if (p.maps == 2 && s == 0 && !zeros) zeros = !__all_sync(0xffffffffu, wait(&ex_full, 0, p.wait)) || *(volatile int*)&cut != 0;
      if (zeros) {
        Vec16<T> zero;
        zero.raw = make_uint4(0, 0, 0, 0);
        if (row_ok && (p.maps == 1 || s == 0))
          for (int k = 0; k < HD; k += 8) st16(out + k, zero);
        ok = false;
      }
      if (p.lse && row_ok)
        p.lse[((int64_t)(t0 + i) * p.H + h) * p.maps + (p.maps == 2 ? s : 0)] = zeros || l == 0.f ? INFINITY : m + log2f(l);
    }
    if (p.splits > 1) {
      float* dst = p.part + ((((int64_t)blockIdx.x * p.splits + blockIdx.y) * 2 + s) * BM + r) * (HD + 2);
      // a wait that ran out: a negative sum, at which the join writes zeros
      *reinterpret_cast<float2*>(dst + HD) = ok ? make_float2(m, l) : make_float2(NONE, -1.f);
#pragma unroll 1
      for (int cc = 0; cc < HD; cc += 32) {
        float o[32];
        if (ntile > 0 && ok) tld32(tl + (uint32_t)(O_COL + s * HD + cc), o);
#pragma unroll
        for (int k = 0; k < 32; k += 2)
          *reinterpret_cast<float2*>(dst + cc + k) = ntile > 0 && ok ? make_float2(o[place(k)], o[place(k + 1)]) : make_float2(0.f, 0.f);
      }
      ok = false;                                  // nothing more to write
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float lam = 0.f, den = 1.f;
    if (p.maps == 2 && row_ok) { lam = p.lam[h]; den = 1.f / (1.f - lam + 1e-8f); }
    float* xrow = reinterpret_cast<float*>(sm) + r * (HD + 4);        // stream B's row; Q and the ring are free now
#pragma unroll 1
    for (int cc = 0; cc < HD && ok; cc += 32) {
      float o[32];
      tld32(tl + (uint32_t)(O_COL + s * HD + cc), o);
#pragma unroll
      for (int k = 0; k < 32; ++k) o[k] *= inv;
      if (p.maps == 2 && s == 1) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(xrow + cc + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
      } else if (row_ok) {
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          Vec16<T> v;
#pragma unroll
          for (int q = 0; q < 8; ++q) v.v[q] = from_f<T>(p.maps == 2 ? (o[place(k + q)] - lam * xrow[cc + place(k + q)]) * den : o[place(k + q)]);
          st16(out + cc + k, v);
        }
      }
    }
    if (p.maps == 2 && s == 1) bar_arrive(&ex_full);
  }
  fence_before();
  __syncthreads();
  if (warp == 8 + NC / 32) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the parts of a row, a warp each: its maps, their splits in order.
template <typename T, int HD>
__global__ void __launch_bounds__(256) chunk_join_kernel(const __grid_constant__ Params p, int units) {
  constexpr int D = HD / 32;
  const Cache4& c = p.c;
  bool odd = false;                                // then there are no parts
  for (int i = threadIdx.x; i < c.B; i += 256) odd = odd || !in_order(c, i);
  if (__syncthreads_or(odd)) return;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (item >= (int64_t)c.T * p.H) return;
  const int t = (int)(item / p.H), h = (int)(item % p.H), g = h / p.rep;
  const int b = sequence_of(c.cu, c.B, t);
  if (b < 0) return;
  const int t0 = c.cu[b], n = c.cu[b + 1] - t0;
  if (!in_order(c, b) || (int64_t)n * p.rep * p.maps <= p.few) return;
  const int rows = p.maps == 2 ? BM : 2 * BM, row = (t - t0) * p.rep + h % p.rep;
  const int u = (int)((int64_t)t0 * p.rep / rows + b) + row / rows;
  const int64_t unit = (int64_t)(units - 1 - u) * c.G + g;
  float res[D] = {};
  for (int map = 0; map < p.maps; ++map) {
    const int s = p.maps == 2 ? map : row % rows / BM;
    const float* x = p.part + ((unit * p.splits * 2 + s) * BM + row % BM) * (HD + 2);
    const int64_t step = (int64_t)2 * BM * (HD + 2);
    float M = NONE, L = 0.f, a[D] = {};
    float least = 0.f;                             // negative where a part was cut short
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i, x += step) {
      const float2 ml = *reinterpret_cast<const float2*>(x + HD);
      least = fminf(least, ml.y);
      float2 v[D / 2];
#pragma unroll
      for (int d = 0; d < D / 2; ++d) v[d] = *reinterpret_cast<const float2*>(x + lane * D + 2 * d);
      const float mn = fmaxf(M, ml.x), f = ex2(M - mn), e = ex2(ml.x - mn);
      M = mn;
      L = fmaf(L, f, ml.y * e);
#pragma unroll
      for (int d = 0; d < D / 2; ++d) {
        a[2 * d] = fmaf(a[2 * d], f, v[d].x * e);
        a[2 * d + 1] = fmaf(a[2 * d + 1], f, v[d].y * e);
      }
    }
    if (p.lse && lane == 0) p.lse[item * p.maps + map] = L == 0.f ? INFINITY : M + log2f(L);
    if (least < 0.f) {                             // of either map: the row is zeros
      __syncwarp();
      if (p.lse && lane < p.maps) p.lse[item * p.maps + lane] = INFINITY;
#pragma unroll
      for (int d = 0; d < D; ++d) res[d] = 0.f;
      break;
    }
    float w = L == 0.f ? 0.f : 1.f / L;
    if (p.maps == 2) w *= (map ? -p.lam[h] : 1.f) / (1.f - p.lam[h] + 1e-8f);
#pragma unroll
    for (int d = 0; d < D; ++d) res[d] = fmaf(a[d], w, res[d]);
  }
  T* out = (T*)p.out + item * HD + lane * D;
#pragma unroll
  for (int d = 0; d < D; ++d) out[d] = from_f<T>(res[d]);
}

template <typename T, int HD>
void launch(const Attn4& attn) {
  auto fn = chunk_kernel<T, HD>;
  Params p;
  static_cast<Attn4&>(p) = attn;
  MAMF_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HD>()));
  const int64_t rows = p.maps == 2 ? BM : 2 * BM;
  const int64_t units = ((int64_t)p.c.T * p.rep / rows + p.c.B) * p.c.G;
  TORCH_CHECK(units < (1LL << 31), "paged_attention: sizes");
  // One CTA runs per SM.  Where the tiles leave SMs idle, several CTAs share the keys of a tile, each at least 8
  // key tiles of the longest sequence that the block table has room for.
  const int64_t longest = ((int64_t)p.c.W * p.c.page + BN - 1) / BN;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({num_sms() / units, longest / 8, 32}));
  at::Tensor ws;
  p.part = nullptr;
  if (p.splits > 1) {
    ws = at::empty({units * p.splits * 2 * BM * (HD + 2)}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA));
    p.part = ws.data_ptr<float>();
  }
  fn<<<dim3((unsigned)units, (unsigned)p.splits), NT, smem_bytes<HD>(), stream()>>>(p);
  MAMF_LAUNCH_CHECK();
  if (p.splits > 1) {
    chunk_join_kernel<T, HD><<<(unsigned)(((int64_t)p.c.T * p.H + 7) / 8), 256, 0, stream()>>>(p, (int)(units / p.c.G));
    MAMF_LAUNCH_CHECK();
  }
}

// ---- received weights ------------------------------------------------------------------------------
// mass[slot] += sum over rows of 2^(score - log2 of the row's sum): the scores once more, transposed, so that a thread sums
// one slot's weights in a register and nothing is added up across threads or CTAs.
//
// rows_kernel lays the rows of q out once: tiles of 128 rows of a sequence and KV head as f16 in the order of the products'
// operand, and behind each tile what a weight needs of its row, {factor, factor, -log2 sum, -log2 sum} of two rows.
// weights_kernel: a CTA holds 256 slots of a KV head as two M = 128 operands, S^T = K Q^T, decoded once into shared memory;
// the tiles with rows that see some of them pass by as N = 128.  10 warps:
//   warps 0-3, 4-7  128 slots each (thread = slot = TMEM lane): S^T from TMEM, a fused multiply-add and an exponential a
//                   weight, two at a time
//   warp 8          one lane copies tiles into a ring of three
//   warp 9          TMEM allocation, MMA issue; two accumulators for each half, so that the sums do not wait for a product
// 256 slots rather than 128: each tile of rows is read from the L2 half as often.  The exponentials alone, 16 a cycle and SM,
// are 2,048 cycles for 256 slots and 128 rows; it takes twice that (4 x 1024 tokens on 7168 cached, one map of 32 / 8 heads:
// 560 us, exponentials 49%, tensor pipe 23%, 31% of the issue slots).  Probably the two summing warps a scheduler are too few to
// hide a load from tensor memory, fused multiply-adds and exponentials one after another; and the keys are decoded before
// the first product.
constexpr int WR = 128, WK = 256, WQ = 3, NTW = 320;       // rows of a tile, slots of a CTA, ring
template <int HD> constexpr int TILE_BYTES = WR * HD * 2 + WR * 8;
template <int HD> constexpr int weights_smem() { return 1024 + WK * HD * 2 + WQ * ((TILE_BYTES<HD> + 1023) / 1024 * 1024); }

struct Weights : Attn4 {
  uint8_t* tiles;            // [unit * G + head][TILE_BYTES]
  int kept;                  // sequences of up to this many rows are not taken
};
// Tiles of sequence b begin at unit cu[b] per / WR + b: it has ceil(n per / WR) or less.
__device__ __forceinline__ int64_t first_unit(const Table& c, int b, int per) { return (int64_t)c.cu[b] * per / WR + b; }
__device__ __forceinline__ bool takes(const Weights& p, int b) {
  if (!in_order(p.c, b)) return false;
  const int64_t rows = (int64_t)(p.c.cu[b + 1] - p.c.cu[b]) * p.rep * p.maps;
  return rows > p.kept && (rows <= p.few || p.chunked);
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ Weights p) {
  constexpr int LANES = HD / 8;                            // of a row, 8 dims each
  const Cache4& c = p.c;
  const int per = p.rep * p.maps, g = blockIdx.y;
  int b = 0;
  for (int hi = c.B - 1; b < hi;) {
    const int mid = (b + hi + 1) >> 1;
    if (first_unit(c, mid, per) <= (int64_t)blockIdx.x) b = mid; else hi = mid - 1;
  }
  if (!takes(p, b)) return;
  const int t0 = c.cu[b];
  const int64_t rows = (int64_t)(c.cu[b + 1] - t0) * per, row0 = ((int64_t)blockIdx.x - first_unit(c, b, per)) * WR;
  if (row0 < 0 || row0 >= rows) return;
  uint8_t* tile = p.tiles + ((int64_t)blockIdx.x * c.G + g) * TILE_BYTES<HD>;
  float* facts = reinterpret_cast<float*>(tile + WR * HD * 2);
  const int k = threadIdx.x % LANES, i0 = (int)(row0 / per), k0 = (int)(row0 % per);      // the first row's token, its place there
  constexpr int STEPS = WR * LANES / 256;
  Vec16<T> x[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int r = (s * 256 + threadIdx.x) / LANES, i = i0 + (k0 + r) / per, j = (k0 + r) % per, h = g * p.rep + j / p.maps;
    x[s].raw = make_uint4(0, 0, 0, 0);
    if (row0 + r < rows)
      x[s] = ld16(j % p.maps ? (const T*)p.q2 + (int64_t)(t0 + i) * p.st2 + (int64_t)h * p.sh2 + 8 * k
                             : (const T*)p.q1 + (int64_t)(t0 + i) * p.st1 + (int64_t)h * p.sh1 + 8 * k);
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int r = (s * 256 + threadIdx.x) / LANES;
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(to_f(x[s].v[e])));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    int e = (int)(__float_as_uint(mx) >> 23) - 127;        // as in the attention
    if (e == -127 || e == 128) e = 0;
    e = max(-126, min(126, e));
    const float down = pow2(-e);
    uint4 v;
    v.x = h2(to_f(x[s].v[0]) * down, to_f(x[s].v[4]) * down);
    v.y = h2(to_f(x[s].v[1]) * down, to_f(x[s].v[5]) * down);
    v.z = h2(to_f(x[s].v[2]) * down, to_f(x[s].v[6]) * down);
    v.w = h2(to_f(x[s].v[3]) * down, to_f(x[s].v[7]) * down);
    *reinterpret_cast<uint4*>(tile + (k >> 3) * (WR * 128) + r * 128 + (((k & 7) ^ (r & 7)) << 4)) = v;
    if (k == 0) {
      facts[(r >> 1) * 4 + (r & 1)] = p.scale_log2 * pow2(e);
      facts[(r >> 1) * 4 + (r & 1) + 2] = row0 + r < rows ? -p.lse[(int64_t)(t0 + i0 + (k0 + r) / per) * p.H * p.maps + g * per + (k0 + r) % per] : -INFINITY;
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(NTW, 1) weights_kernel(const __grid_constant__ Weights p) {
  constexpr int KB2 = WR * HD * 2, STAGE = (TILE_BYTES<HD> + 1023) / 1024 * 1024;       // bytes of 128 slots, of a ring's place
  const Cache4& c = p.c;
  const int g = blockIdx.y, b = blockIdx.z, base = blockIdx.x * WK, per = p.rep * p.maps;
  const int len = cached_length(c, c.lens[b]);
  if (base >= len || !takes(p, b)) return;
  bool odd = false;                                        // offsets out of order anywhere: not all tiles are there
  for (int i = threadIdx.x; i < c.B; i += NTW) odd = odd || !in_order(c, i);
  if (__syncthreads_or(odd)) return;
  const int n = c.cu[b + 1] - c.cu[b], at0 = len - n;
  const int64_t rows = (int64_t)n * per;
  // tokens [i0, i1) see some slot of the CTA's
  const int i0 = max(0, base - at0), last = min(base + WK, len) - 1;
  const int i1 = p.window > 0 ? (int)min((int64_t)n, (int64_t)last + p.window - at0) : n;
  if (i0 >= i1) return;
  // The first slot that some row of the sequence sees.  A page below it may be another sequence's by now, whose CTA is adding
  // to its weights: it is not touched, not even to add 0.
  const int seen = p.window > 0 ? max(0, at0 - p.window + 1) : 0;
  const int64_t j0 = (int64_t)i0 * per / WR;
  const int ntile = (int)(((int64_t)i1 * per + WR - 1) / WR - j0);
  const uint8_t* tiles = p.tiles + ((first_unit(c, b, per) + j0) * c.G + g) * TILE_BYTES<HD>;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sm + 2 * KB2;
  __shared__ uint64_t q_full[WQ], q_empty[WQ], s_full[4], s_empty[4], idle;
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < WQ; ++i) { bar_init(&q_full[i], 1); bar_init(&q_empty[i], 9); }
    for (int i = 0; i < 4; ++i) { bar_init(&s_full[i], 1); bar_init(&s_empty[i], 128); }
    bar_init(&idle, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // keys: a 16-byte chunk of codes (32 dims) per thread and turn; slots that nobody sees, or of no page, become zeros
  for (int i = threadIdx.x; i < WK * (HD / 32); i += NTW) {
    const int tok = i / (HD / 32), cc = i % (HD / 32), slot = base + tok;
    uint4 x = make_uint4(0, 0, 0, 0);
    uint32_t params[HD / 64] = {};
    if (slot >= seen && slot < len) {
      const int pg = c.table[(int64_t)b * c.W + (slot >> c.shift)];
      if (pg >= 0 && pg < c.P) {
        const uint8_t* blk = block_of<HD>(c, pg, g, slot);
        x = *reinterpret_cast<const uint4*>(blk + (tok & 15) * (HD / 2) + cc * 16);
#pragma unroll
        for (int k = 0; k < HD / 64; ++k) params[k] = reinterpret_cast<const uint32_t*>(blk + PARAMS<HD> + (tok & 15) * (HD / 16))[k];
      }
    }
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint8_t* row = sm + (tok >> 7) * KB2 + (cc >> 1) * (WR * 128) + (tok & 127) * 128;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      uint32_t h[4];
      decode(w[m], levels_of(params[HD == 128 ? m & 1 : 0], c.base), c.base, h);
      *reinterpret_cast<uint4*>(row + ((((cc & 1) * 4 + m) ^ (tok & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
  fence_async_smem();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 8) {
    // ------------------------------- rows -------------------------------
    if (lane == 0) {
      bool ok = true;
      int j = 0;
      for (; j < ntile; ++j) {
        const int st = j % WQ;
        if (j >= WQ) ok = wait(&q_empty[st], (uint32_t)((j / WQ - 1) & 1), p.wait);
        if (!ok) break;
        bar_expect_tx(&q_full[st], TILE_BYTES<HD>);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(su32(ring + st * STAGE)), "l"(tiles + (int64_t)j * c.G * TILE_BYTES<HD>), "r"(TILE_BYTES<HD>), "r"(su32(&q_full[st])) : "memory");
      }
      // after a wait that ran out: the copies that are still under way into this CTA's memory
      if (!ok)
        for (int k = max(0, j - WQ); k < j; ++k)
          for (const long long t = clock64(); !try_once(&q_full[k % WQ], (uint32_t)((k / WQ) & 1)) && clock64() - t <= WAIT_CYCLES;) {}
    }
  } else if (warp == 9) {
    // ------------------------------- MMA issue -------------------------------
    if (lane == 0) {
      constexpr uint32_t ID = idesc(WR, false);
      bool ok = true;
      for (int j = 0; j < ntile && ok; ++j) {
        const int st = j % WQ;
        ok = wait(&q_full[st], (uint32_t)((j / WQ) & 1), p.wait);
        const uint32_t qb = su32(ring + st * STAGE);
        for (int s = 0; s < 2 && ok; ++s) {
          const int buf = 2 * s + (j & 1);
          if (j >= 2) ok = wait(&s_empty[buf], (uint32_t)((j / 2 - 1) & 1), p.wait);
          if (!ok) break;
          fence_after();
          const uint32_t ka = su32(sm + s * KB2);
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            mma_ss(tmem + (uint32_t)(buf * WR), sdesc(ka + (k >> 2) * (WR * 128) + (k & 3) * 32, 16, 1024),
                   sdesc(qb + (k >> 2) * (WR * 128) + (k & 3) * 32, 16, 1024), ID, k > 0 ? 1u : 0u);
          commit(&s_full[buf]);
        }
        if (ok) commit(&q_empty[st]);
      }
      // products under way read shared memory and write TMEM, both of which go when the CTA ends
      commit(&idle);
      for (const long long t = clock64(); !try_once(&idle, 0) && clock64() - t <= WAIT_CYCLES;) {}
    }
  } else {
    // ------------------------------- sums -------------------------------
    const int s = warp >> 2, r = (warp & 3) * 32 + lane, from = base + s * WR, slot = from + r;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
    bool ok = true;
    for (int j = 0; j < ntile && ok; ++j) {
      const int st = j % WQ, buf = 2 * s + (j & 1);
      // the tile's facts, too, are there
      ok = __all_sync(0xffffffffu, wait(&q_full[st], (uint32_t)((j / WQ) & 1), p.wait) && wait(&s_full[buf], (uint32_t)((j >> 1) & 1), p.wait));
      if (!ok) break;
      fence_after();
      const int64_t row0 = (j0 + j) * WR;
      const int low = at0 + (int)(row0 / per), high = at0 + (int)((min(row0 + WR, rows) - 1) / per);
      const bool all = from + WR - 1 <= low && (p.window == 0 || from > high - p.window);
      const float* fact = reinterpret_cast<const float*>(ring + st * STAGE + KB2);
#pragma unroll 1
      for (int cc = 0; cc < WR; cc += 32) {
        float v[32];
        tld32(tl + (uint32_t)(buf * WR + cc), v);
        if (cc == WR - 32) {                               // the accumulator is read
          fence_before();
          bar_arrive(&s_empty[buf]);
        }
        // two loops: a question inside the one would put its pairs behind one another
        if (all) {
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float4 f = *reinterpret_cast<const float4*>(fact + 2 * (cc + k));
            float e0, e1;
            unpk(fma2(pk(v[k], v[k + 1]), pk(f.x, f.y), pk(f.z, f.w)), e0, e1);
            sum[k / 2 & 3] = add2(sum[k / 2 & 3], pk(ex2(e0), ex2(e1)));
          }
        } else {
          int at = at0 + (int)((row0 + cc) / per), of = (int)((row0 + cc) % per);      // the row's slot, its place in its token
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float f = fact[4 * ((cc + k) >> 1) + (k & 1)], minus = fact[4 * ((cc + k) >> 1) + (k & 1) + 2];
            const float e = slot > at || (p.window > 0 && slot <= at - p.window) ? 0.f : ex2(fmaf(v[k], f, minus));
            sum[k & 3] = add2(sum[k & 3], pk(e, 0.f));
            ++of;
            at += of == per;
            of = of == per ? 0 : of;
          }
        }
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&q_empty[st]);
    }
    float a, a2;
    unpk(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, a2);
    if (ok && slot >= seen && slot < len) {
      const int pg = c.table[(int64_t)b * c.W + (slot >> c.shift)];
      if (pg >= 0 && pg < c.P) c.mass[(((int64_t)pg * c.G + g) << c.shift) + (slot & (c.page - 1))] += a + a2;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <typename T, int HD>
void launch_weights(const Attn4& attn, int kept) {
  Weights p;
  static_cast<Attn4&>(p) = attn;
  p.kept = kept;
  const int64_t units = (int64_t)p.c.T * p.rep * p.maps / WR + p.c.B;
  TORCH_CHECK(units < (1LL << 31), "paged_attention: sizes");
  const at::Tensor ws = at::empty({units * p.c.G * TILE_BYTES<HD>}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA));
  p.tiles = ws.data_ptr<uint8_t>();
  rows_kernel<T, HD><<<dim3((unsigned)units, (unsigned)p.c.G), 256, 0, stream()>>>(p);
  MAMF_LAUNCH_CHECK();
  auto fn = weights_kernel<T, HD>;
  MAMF_CUDA_CHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, weights_smem<HD>()));
  const int64_t tiles = ((int64_t)p.c.W * p.c.page + WK - 1) / WK;
  fn<<<dim3((unsigned)tiles, (unsigned)p.c.G, (unsigned)p.c.B), NTW, weights_smem<HD>(), stream()>>>(p);
  MAMF_LAUNCH_CHECK();
}

}  // namespace ptc4

namespace paged4 {
void chunk_weights(const Attn4& p, int kept, int hd, bool bf16) {
  if (bf16) { if (hd == 128) ptc4::launch_weights<__nv_bfloat16, 128>(p, kept); else ptc4::launch_weights<__nv_bfloat16, 64>(p, kept); }
  else { if (hd == 128) ptc4::launch_weights<__half, 128>(p, kept); else ptc4::launch_weights<__half, 64>(p, kept); }
}
void chunk_attention(const Attn4& p, int hd, bool bf16) {
  if (bf16) { if (hd == 128) ptc4::launch<__nv_bfloat16, 128>(p); else ptc4::launch<__nv_bfloat16, 64>(p); }
  else { if (hd == 128) ptc4::launch<__half, 128>(p); else ptc4::launch<__half, 64>(p); }
}
int64_t chunk_error(bool clear) { return take_code(ptc4::g_err, clear) | take_code(ptc4::g_wait_err, clear); }
}  // namespace paged4

}  // namespace mamf
