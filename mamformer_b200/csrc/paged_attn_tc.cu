// Attention over the paged 8-bit cache (layout in paged.cuh) for many query rows per KV head: chunks of a
// prompt.  The products run on the 5th-generation tensor cores; every key tile is read once per CTA.
//
// A CTA holds two streams of 128 query rows of one KV head that share its keys and values:
//   differential: the two maps of the same rows;   single softmax: two neighbouring tiles of rows.
// A row is (token, head of the group), so short runs of tokens still fill a tile.  11 warps:
//   warps 0-3, 4-7  softmax of stream A, B (thread = row = TMEM lane): write the row of q to shared memory
//                   as f16, scaled by a power of two to [1, 2); then S from TMEM, P as packed f16 back over it
//   warps 8-9       keys and values: 64-token tiles, 16 bytes per load, through registers one tile ahead,
//                   e4m3 -> f16 (exact) into a ring of 128-byte-swizzled tiles; codes past the end become 0
//   warp 10         TMEM allocation, MMA issue: S = Q K^T (M 128, N 64), O += P V (N = head size, P in TMEM)
// The blocks' scales are powers of two and stay out of the products: a key's goes into the factor of its
// score, a value's into the exponent of its weight.  O is kept in units of 2^(m + r): m is the row's running maximum of
// the scores, which the sum of weights is kept in, and r a whole number that brings m + r to its running maximum of
// score + log2 of the value scale.  So the f16 weights keep their bits for what the row sees, whatever the values of
// other pages are, and the largest score's is a power of two.  A 16-token group costs a handful of operations per row.
// Where there are fewer tiles than SMs, several CTAs share a tile's keys and a second kernel joins them.  Online softmax
// with lazy rescaling as in flash_tc.cu.  Every wait is bounded; a wait that runs out records a code, and the CTA winds
// down and leaves zeros.
//
// P is rounded to f16: 11 bits of a weight, where bf16 would keep 8, and a second product for the lower bits would be half
// of the tensor work again; its sum is fp32.  In bf16 the result's own rounding hides it; f16 results of short runs are 2.9e-4
// from 64 bits, 2.1e-4 with fp32 arithmetic.
//
// 2 x 2048 tokens on 10240 cached, 32 / 8 heads of 128, two maps: 1.74 ms, 871 TFLOP/s.  A pair of tiles takes
// 2,670 cycles; the products' own time is 1,024.  It is bound by the hand-offs: the products of the scores
// take 70-80 cycles each (32 at the full rate, N = 64), those of the values 160-190 (64), and a tile's
// conversion 1,130 with 1,550 until the next one's loads are there; without the exponentials it is as slow.
#include "f32x2.cuh"
#include "paged.cuh"
#include "tc5.cuh"

namespace mamf {
namespace ptc {

using namespace paged;
using namespace tc5;

constexpr int BM = 128, BN = 64, ST = 4, NC = 64, NT = 256 + NC + 32;       // NC converting threads
constexpr float LAZY = 8.f, NONE = -1e30f;

__device__ int g_err = 0, g_wait_err = 0;

template <int HD> constexpr int q_bytes() { return BM * HD * 2; }
template <int HD> constexpr int k_bytes() { return BN * HD * 2; }
// the epilogue's exchange rows (fp32) lie over Q and the ring
template <int HD> constexpr int smem_bytes() { return 1024 + 2 * q_bytes<HD>() + 2 * ST * k_bytes<HD>(); }

struct Params : Attn {
  int splits;          // CTAs that share a tile's keys; with more than one they leave parts for the join kernel:
  float* part;         // [unit * G + head][split][stream][BM][HD + 2]: O (not divided), m, l
};

// As tc5::bar_wait, without its suspend-time hint: the hand-offs of a tile are short (1.72 ms against 1.77).  The error
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
__device__ __forceinline__ void to_h4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// What the softmax needs to know of a tile's four 16-token groups.
struct __align__(16) Groups {
  float k[4];          // scale of the keys, 0: the group is not there
  float v[4];          // log2 of the scale of the values
  float c[4];          // 1 / scale of the values
  int all;             // all four groups are there
};

template <typename T, int HD>
__global__ void __launch_bounds__(NT, 1) chunk_kernel(const __grid_constant__ Params p) {
  constexpr int QB = q_bytes<HD>(), KB = k_bytes<HD>();
  constexpr int O_COL = 256;                       // TMEM: S_A[2], S_B[2] of 64 columns, then O_A, O_B of HD
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t q_full, kv_full[ST], kv_empty[ST], s_full[4], p_full[4], o_done[4], ex_full, idle;
  __shared__ Groups groups[ST];
  __shared__ uint32_t tmem_slot;
  __shared__ int cut;                              // a wait of the second map ran out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cache& c = p.c;

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
      if (__syncthreads_or(odd)) {                 // no unit may have some rows: none of the call's results count
        for (int64_t i = threadIdx.x; i < c.T * row; i += NT) ((T*)p.out)[i] = from_f<T>(0.f);
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
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  uint8_t* ring = sm + 2 * QB;

  if (warp >= 8 && warp < 8 + NC / 32) {
    // ------------------------------- keys and values -------------------------------
    constexpr int CR = HD / 16, N = BN * CR / NC;           // 16-byte chunks of a token, chunks per thread
    constexpr int RS = NC / CR;                              // rows between a thread's chunks: 8 or 16
    const int ct = threadIdx.x - 256, r0c = ct / CR, cc = ct % CR;
    uint4 kx[N], vx[N];                                      // chunk i: token i RS + r0c, dims 16 cc ..
    float ks = 0.f, vs = 0.f;                                // of group lane % 4
    auto look_up = [&](int j) {                              // the page of group lane % 4 of tile j
      const int slot = (kt0 + j) * BN + (lane & 3) * 16;
      if (j >= ntile || slot >= key_hi || slot + 16 <= key_lo) return -2;      // nothing to see there: no page is asked for
      const int w = slot >> c.shift;
      const int pg = w < c.W ? c.table[(int64_t)b * c.W + w] : -1;
      return (unsigned)pg < (unsigned)c.P ? pg : -1;
    };
    auto load = [&](int j, int pg) {
      const int slot = (kt0 + j) * BN;
      const int64_t blk = (int64_t)pg * c.G + g;
      ks = vs = 0.f;
      if (pg >= 0) { ks = c.ks[blk]; vs = c.vs[blk]; }
      else if (pg == -1 && ct < 4) atomicCAS(&g_err, 0, (int)ERR_PAGE);
      // byte offset of the group's first token, -1: not there
      const int64_t mine = pg >= 0 ? ((blk << c.shift) + ((slot + (lane & 3) * 16) & (c.page - 1))) * HD : -1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t off = __shfl_sync(0xffffffffu, mine, q) + r0c * HD + cc * 16;
        const bool there = __shfl_sync(0xffffffffu, pg, q) >= 0;
#pragma unroll
        for (int i = q * 16 / RS; i < (q + 1) * 16 / RS; ++i) {
          kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
          if (there && slot + i * RS + r0c < key_hi) {       // codes past the end may be anything, NaN included
            kx[i] = *reinterpret_cast<const uint4*>(c.k + off + (i * RS - q * 16) * HD);
            vx[i] = *reinterpret_cast<const uint4*>(c.v + off + (i * RS - q * 16) * HD);
          }
        }
      }
    };
    // place of chunk 0's two 16-byte halves; row i RS + r0c has the same place in its 8 rows of 128 bytes.
    // The lanes of the second 64 dims store their halves the other way round: the banks of both differ.
    const int c0 = ((cc & 3) * 2) ^ (r0c & 7), swap = cc >> 2 & 1;
    uint8_t* const at = ring + (cc >> 2) * (BN * 128) + r0c * 128;
    const int first = (c0 ^ swap) * 16, second = (c0 ^ swap ^ 1) * 16;
    auto store = [&](uint8_t* row, const uint4& x) {
      uint4 lo, hi;
      to_h4(x.x, lo.x, lo.y);
      to_h4(x.y, lo.z, lo.w);
      to_h4(x.z, hi.x, hi.y);
      to_h4(x.w, hi.z, hi.w);
      *reinterpret_cast<uint4*>(row + first) = swap ? hi : lo;
      *reinterpret_cast<uint4*>(row + second) = swap ? lo : hi;
    };
    if (ntile > 0) load(0, look_up(0));
    int next = look_up(1);
    bool ok = true;
    for (int j = 0; j < ntile; ++j) {
      const int st = j % ST;
      if (j >= ST) ok = __all_sync(0xffffffffu, wait(&kv_empty[st], (uint32_t)((j / ST - 1) & 1), p.wait));
      if (!ok) break;
      const bool all = __all_sync(0xffffffffu, ks != 0.f);
      if (ct < 4) {
        const int e = vs > 0.f ? (int)(__float_as_uint(vs) >> 23) - 127 : 0;
        groups[st].k[ct] = ks;
        groups[st].v[ct] = (float)e;
        groups[st].c[ct] = pow2(max(-126, -e));
        if (ct == 0) groups[st].all = all;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        store(at + st * 2 * KB + i * RS * 128, kx[i]);
        store(at + st * 2 * KB + KB + i * RS * 128, vx[i]);
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
        v.x = h2(to_f(x[k].v[0]) * down, to_f(x[k].v[1]) * down);
        v.y = h2(to_f(x[k].v[2]) * down, to_f(x[k].v[3]) * down);
        v.z = h2(to_f(x[k].v[4]) * down, to_f(x[k].v[5]) * down);
        v.w = h2(to_f(x[k].v[6]) * down, to_f(x[k].v[7]) * down);
        *reinterpret_cast<uint4*>(qrow + (k >> 3) * (BM * 128) + (((k & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_async_smem();
      bar_arrive(&q_full);
    }
    // slots [lo, hi] that the row sees; rows past the last one (zeros) see everything and are not written
    const int hi = row_ok ? min(len - 1, at) : 0x7fffffff, lo = row_ok && p.window > 0 ? at - p.window + 1 : 0;
    float m = NONE, r2 = 0.f, unit = 1.f, l = 0.f;           // r2: r of the head comment;  unit = 2^r2
    bool ok = true;
    for (int j = 0; j < ntile && ok; ++j) {
      const int buf = j & 1, st = j % ST;
      ok = __all_sync(0xffffffffu, wait(&kv_full[st], (uint32_t)((j / ST) & 1), p.wait) && wait(&s_full[s * 2 + buf], (uint32_t)((j >> 1) & 1), p.wait));
      if (!ok) break;
      fence_after();
      float sv[BN];
      tld64(tl + (uint32_t)(s * 128 + buf * 64), sv);
      const Groups& gr = groups[st];
      float f[4];
      *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(gr.k);
      const int kbase = (kt0 + j) * BN;
      if (__any_sync(0xffffffffu, !(gr.all && kbase >= lo && kbase + BN - 1 <= hi))) {
#pragma unroll
        for (int k = 0; k < BN; ++k) {
          const int key = kbase + k;
          sv[k] = (key >= lo && key <= hi && f[k >> 4] != 0.f) ? sv[k] : -INFINITY;
        }
        // a factor that is 0, or underflows, would make a masked score's -inf NaN; products are below 2^18, so that this
        // one's scores are 0 all the same
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = fmaxf(f[k] * rs, 1e-37f);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] *= rs;
      }
      float mx = -INFINITY, vx = -INFINITY;
      float gv[4];
      *reinterpret_cast<float4*>(gv) = *reinterpret_cast<const float4*>(gr.v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) a[q] = fmaxf(fmaxf(sv[16 * k + q], sv[16 * k + 4 + q]), fmaxf(sv[16 * k + 8 + q], sv[16 * k + 12 + q]));
        a[0] = fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * f[k];
        mx = fmaxf(mx, a[0]);
        vx = fmaxf(vx, a[0] + gv[k]);
      }
      float fo = 1.f;
      if (mx > m + LAZY || vx > m + r2 + LAZY) {            // both rise once one of them is outgrown
        const float m1 = fmaxf(m, mx), r1 = rintf(fmaxf(vx, m + r2) - m1);
        l *= ex2(m - m1);                                   // 0 for the first key of a row
        fo = ex2((m - m1) + (r2 - r1));
        m = m1;
        r2 = r1;
        unit = pow2((int)fminf(fmaxf(r1, -126.f), 126.f));
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
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // Weights of a group whose scale is below 2^-60 of the reference enter as if it were that, which is as little
        // as nothing in O; this keeps them, and so their sum for l, in range.
        const float neg = fmaxf(gv[k] - r2, -60.f) - m;
        const uint64_t ff = pk(f[k], f[k]), nn = pk(neg, neg);
        uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float e0, e1;
          unpk(fma2(pk(sv[16 * k + 2 * q], sv[16 * k + 2 * q + 1]), ff, nn), e0, e1);
          e0 = ex2(e0);
          e1 = ex2(e1);
          sum[q & 1] = add2(sum[q & 1], pk(e0, e1));
          pk_[8 * k + q] = __uint_as_float(h2(e0, e1));
        }
        float a, a2;
        unpk(add2(sum[0], sum[1]), a, a2);
        l = fmaf(a + a2, fminf(gr.c[k] * unit, 1.1529215e18f), l);         // 2^60
      }
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
          *reinterpret_cast<float2*>(dst + cc + k) = ntile > 0 && ok ? make_float2(o[k] * unit, o[k + 1] * unit) : make_float2(0.f, 0.f);
      }
      ok = false;                                  // nothing more to write
    }
    const float inv = l == 0.f ? 0.f : unit / l;
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
          for (int q = 0; q < 8; ++q) v.v[q] = from_f<T>(p.maps == 2 ? (o[k + q] - lam * xrow[cc + k + q]) * den : o[k + q]);
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
  const Cache& c = p.c;
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
    if (least < 0.f) {                             // of either map: the row is zeros
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
void launch(const Attn& attn) {
  auto fn = chunk_kernel<T, HD>;
  Params p;
  static_cast<Attn&>(p) = attn;
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

}  // namespace ptc

namespace paged {
void paged_chunk_attention(const Attn& p, int hd, bool bf16) {
  if (bf16) { if (hd == 128) ptc::launch<__nv_bfloat16, 128>(p); else ptc::launch<__nv_bfloat16, 64>(p); }
  else { if (hd == 128) ptc::launch<__half, 128>(p); else ptc::launch<__half, 64>(p); }
}
int64_t paged_chunk_error(bool clear) { return take_code(ptc::g_err, clear) | take_code(ptc::g_wait_err, clear); }
}  // namespace paged

}  // namespace mamf
